// The training-step operators on torch tensors: checks, outputs, workspaces, the call into the C ABI (gsa_b200.h) on the
// tensors' device and its current stream, and the autograd functions.  The same division of labour as gsa_b200/ops.py
// (the ABI allocates nothing and sees raw pointers), in C++ because a step makes many such calls on small tensors: a call
// costs the host a third of what it does through ctypes, and a backward pass needs no interpreter.
//
// The library's entry points are handed in by the Python package (bind), which loads it; nothing here links to it.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/extension.h>

#include <algorithm>
#include <functional>
#include <numeric>
#include <optional>
#include <tuple>
#include <vector>

#include "gsa_b200.h"

namespace py = pybind11;
using at::Tensor;
using std::optional;

namespace {

struct Api {
  decltype(&gsa_rotary) rotary;
  decltype(&gsa_pack_e4m3) pack;
  decltype(&gsa_unpack_e4m3) unpack;
  decltype(&gsa_silu_mul_pack) silu_mul_pack;
  decltype(&gsa_silu_mul_packed_backward) silu_mul_bwd;
  decltype(&gsa_add_rmsnorm_pack) norm_pack;
  decltype(&gsa_rmsnorm_packed_workspace_size) norm_ws;
  decltype(&gsa_rmsnorm_packed_backward) norm_bwd;
  decltype(&gsa_next_token_loss) loss;
  decltype(&gsa_next_token_loss_workspace_size) loss_ws;
  decltype(&gsa_scale) scale;
} api;

// A nonzero status of an entry point; becomes gsa_b200._lib.GSAError.
struct Status : std::runtime_error {
  const char* fn;
  int status;
  Status(const char* f, int s) : std::runtime_error(std::string(f) + " failed with status " + std::to_string(s)), fn(f), status(s) {}
};
void ok(const char* fn, int status) {
  if (status != GSA_OK) throw Status(fn, status);
}

// The tensor's device made current, with its current stream.
struct On {
  c10::cuda::CUDAGuard guard;
  gsa_stream_t stream;
  explicit On(const Tensor& t)
      : guard(t.device()), stream(reinterpret_cast<gsa_stream_t>(c10::cuda::getCurrentCUDAStream(t.get_device()).stream())) {}
};

int code_of(at::ScalarType t) {
  if (t == at::kFloat) return GSA_DTYPE_F32;
  TORCH_CHECK_NOT_IMPLEMENTED(t == at::kBFloat16, "GSA B200 kernels support float32 and bfloat16, got ", t);
  return GSA_DTYPE_BF16;
}

void on_gpu(const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "GSA B200 ops take CUDA tensors only (there is no CPU path)");
}
void beside(const Tensor& t, const Tensor& like) {
  on_gpu(t);
  TORCH_CHECK_VALUE(t.device() == like.device(), "a tensor is on ", t.device(), ", expected ", like.device());
}
void alike(const Tensor& t, const Tensor& like) {
  beside(t, like);
  TORCH_CHECK_VALUE(t.scalar_type() == like.scalar_type(), "a tensor is ", t.scalar_type(), ", expected ", like.scalar_type());
}
void alike(const optional<Tensor>& t, const Tensor& like) {
  if (t) alike(*t, like);
}

// A forward-mode tangent would be lost: none of the operators passes one on.
void no_tangent(const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), "forward-mode derivatives of the training-step operators are not implemented");
}
void no_tangent(const optional<Tensor>& t) {
  if (t) no_tangent(*t);
}

void* ptr(const Tensor& t) { return t.data_ptr(); }
void* ptr(const optional<Tensor>& t) { return t ? t->data_ptr() : nullptr; }

Tensor fresh(const Tensor& like) { return at::empty(like.sizes(), like.options()); }

// A tensor that the caller hands in to be written: none whose own gradient would then be that of what it held before.
void overwritable(const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(at::GradMode::is_enabled() && t.requires_grad()),
                              "the training-step operators write into tensors without autograd only");
}
// A tensor that the caller handed in has been written: graphs that saved it notice.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

int64_t rows_of(at::IntArrayRef shape) {  // all but the last dimension
  int64_t n = 1;
  for (size_t i = 0; i + 1 < shape.size(); ++i) n *= shape[i];
  return n;
}
// t [..., n] as [rows, n] with contiguous values: a view where its strides allow one.
Tensor as_rows(const Tensor& t) {
  const int64_t n = t.size(-1);
  Tensor r = t.dim() == 2 ? t : t.reshape({rows_of(t.sizes()), n});
  return n <= 1 || r.stride(1) == 1 ? r : r.contiguous();
}

// -- packed tensors: one buffer of codes, rows padded to 16, then a scale byte for each group of 32 ---------------
struct PackedRows {
  uint8_t* codes;
  uint8_t* scales;
  int64_t c_ld, s_ld;
};
int64_t code_ld(int64_t n) { return (n + 15) / 16 * 16; }
int64_t scale_ld(int64_t n) { return (n + 31) / 32; }
Tensor packed_buffer(const Tensor& like, int64_t rows, int64_t n) {
  return at::empty({rows * (code_ld(n) + scale_ld(n))}, like.options().dtype(at::kByte));
}
PackedRows packed_rows(const Tensor& data, int64_t rows, int64_t n) {
  TORCH_CHECK_VALUE(data.scalar_type() == at::kByte && data.is_contiguous() &&
                        data.numel() == rows * (code_ld(n) + scale_ld(n)),
                    "a packed buffer of ", data.numel(), " bytes does not hold ", rows, " rows of ", n);
  uint8_t* p = data.data_ptr<uint8_t>();
  return {p, p + rows * code_ld(n), code_ld(n), scale_ld(n)};
}

Tensor pack(const Tensor& x) {
  on_gpu(x);
  no_tangent(x);
  TORCH_CHECK_VALUE(x.dim() > 0, "pack_e4m3 takes a tensor with a last dimension");
  const int code = code_of(x.scalar_type());
  const int64_t n = x.size(-1), rows = rows_of(x.sizes());
  const On on(x);
  Tensor data = packed_buffer(x, rows, n);
  if (x.numel() == 0) return data;
  const Tensor r = as_rows(x);
  const PackedRows p = packed_rows(data, rows, n);
  ok("gsa_pack_e4m3", api.pack(code, rows, n, ptr(r), r.stride(0), p.codes, p.c_ld, p.scales, p.s_ld, on.stream));
  return data;
}

Tensor unpack(const Tensor& data, const std::vector<int64_t>& shape, at::ScalarType dtype) {
  on_gpu(data);
  TORCH_CHECK_VALUE(!shape.empty(), "a packed tensor has a last dimension");
  const int code = code_of(dtype);
  const On on(data);
  Tensor x = at::empty(shape, data.options().dtype(dtype));
  const int64_t n = shape.back(), rows = rows_of(shape);
  const PackedRows p = packed_rows(data, rows, n);
  if (x.numel() == 0) return x;
  ok("gsa_unpack_e4m3", api.unpack(code, rows, n, p.codes, p.c_ld, p.scales, p.s_ld, ptr(x), n, on.stream));
  return x;
}

std::tuple<Tensor, Tensor> silu_mul_packed(const Tensor& gu) {
  on_gpu(gu);
  no_tangent(gu);
  TORCH_CHECK_VALUE(gu.dim() > 0 && gu.size(-1) % 2 == 0, "silu_mul_packed takes [..., 2n], got ", gu.sizes());
  const int code = code_of(gu.scalar_type());
  const int64_t n = gu.size(-1) / 2, rows = rows_of(gu.sizes());
  const On on(gu);
  auto shape = gu.sizes().vec();
  shape.back() = n;
  Tensor z = at::empty(shape, gu.options()), data = packed_buffer(gu, 2 * rows, n);
  if (z.numel() == 0) return {z, data};
  const Tensor r = as_rows(gu);
  const PackedRows p = packed_rows(data, 2 * rows, n);
  ok("gsa_silu_mul_pack",
     api.silu_mul_pack(code, rows, n, ptr(r), r.stride(0), ptr(z), n, p.codes, p.c_ld, p.scales, p.s_ld, on.stream));
  return {z, data};
}

std::tuple<Tensor, optional<Tensor>> silu_mul_packed_backward(const Tensor& dz, const Tensor& data, bool want_z) {
  on_gpu(dz);
  no_tangent(dz);
  beside(data, dz);
  TORCH_CHECK_VALUE(dz.dim() > 0, "silu_mul_packed_backward takes [..., n]");
  const int code = code_of(dz.scalar_type());
  const int64_t n = dz.size(-1), rows = rows_of(dz.sizes());
  const On on(dz);
  auto shape = dz.sizes().vec();
  shape.back() = 2 * n;
  Tensor dgu = at::empty(shape, dz.options());
  optional<Tensor> z;
  if (want_z) z = fresh(dz);
  const PackedRows p = packed_rows(data, 2 * rows, n);
  if (dz.numel() == 0) return {dgu, z};
  const Tensor r = as_rows(dz);
  ok("gsa_silu_mul_packed_backward",
     api.silu_mul_bwd(code, rows, n, ptr(r), r.stride(0), p.codes, p.c_ld, p.scales, p.s_ld, ptr(dgu), 2 * n, ptr(z), n,
                      on.stream));
  return {dgu, z};
}

std::tuple<optional<Tensor>, Tensor, Tensor, Tensor> add_rmsnorm_packed(const Tensor& x, const optional<Tensor>& a,
                                                                        const Tensor& weight, double eps) {
  on_gpu(x);
  no_tangent(x);
  no_tangent(a);
  no_tangent(weight);
  TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0 && weight.dim() == 1 && weight.size(0) == x.size(-1) &&
                        (!a || a->sizes() == x.sizes()),
                    "add_rmsnorm_packed: x ", x.sizes(), ", weight ", weight.sizes(),
                    ", and an addend of another shape than x or a weight of another length than its rows");
  alike(a, x);
  alike(weight, x);
  const int code = code_of(x.scalar_type());
  const int64_t d = x.size(-1), rows = rows_of(x.sizes());
  const On on(x);
  optional<Tensor> h;
  if (a) h = fresh(x);
  Tensor y = fresh(x), data = packed_buffer(x, rows, d);
  Tensor rstd = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  if (rows == 0) return {h, y, data, rstd};
  const Tensor xr = as_rows(x), w = weight.contiguous();
  const optional<Tensor> ar = a ? optional<Tensor>(as_rows(*a)) : std::nullopt;
  const PackedRows p = packed_rows(data, rows, d);
  ok("gsa_add_rmsnorm_pack",
     api.norm_pack(code, rows, d, ptr(xr), xr.stride(0), ptr(ar), ar ? ar->stride(0) : 0, ptr(w), (float)eps, ptr(h), d,
                   ptr(y), d, p.codes, p.c_ld, p.scales, p.s_ld, rstd.data_ptr<float>(), on.stream));
  return {h, y, data, rstd};
}

std::tuple<Tensor, optional<Tensor>, optional<Tensor>> rmsnorm_packed_backward(const Tensor& dy, const Tensor& data,
                                                                               const Tensor& rstd, const Tensor& weight,
                                                                               const optional<Tensor>& dh, bool want_y,
                                                                               bool want_dw) {
  on_gpu(dy);
  no_tangent(dy);
  no_tangent(weight);
  no_tangent(dh);
  TORCH_CHECK_VALUE(dy.dim() > 0 && dy.size(-1) > 0 && weight.dim() == 1 && weight.size(0) == dy.size(-1) &&
                        (!dh || dh->sizes() == dy.sizes()) && rstd.sizes() == dy.sizes().slice(0, dy.dim() - 1) &&
                        rstd.scalar_type() == at::kFloat,
                    "rmsnorm_packed_backward: dy ", dy.sizes(), ", weight ", weight.sizes(), ", rstd ", rstd.sizes(),
                    " do not fit one another");
  alike(weight, dy);
  alike(dh, dy);
  beside(data, dy);
  beside(rstd, dy);
  const int code = code_of(dy.scalar_type());
  const int64_t d = dy.size(-1), rows = rows_of(dy.sizes());
  const On on(dy);
  const PackedRows p = packed_rows(data, rows, d);
  Tensor dx = fresh(dy);
  optional<Tensor> y, dw, ws;
  if (want_y) y = fresh(dy);
  if (rows == 0) {
    if (want_dw) dw = at::zeros({d}, dy.options());
    return {dx, dw, y};
  }
  int64_t bytes = 0;
  if (want_dw) {
    dw = at::empty({d}, dy.options());
    bytes = api.norm_ws(rows, d);
    ws = at::empty({bytes}, dy.options().dtype(at::kByte));
  }
  const Tensor dr = as_rows(dy), w = weight.contiguous(), rs = rstd.contiguous();
  const optional<Tensor> hr = dh ? optional<Tensor>(as_rows(*dh)) : std::nullopt;
  ok("gsa_rmsnorm_packed_backward",
     api.norm_bwd(code, rows, d, ptr(dr), dr.stride(0), ptr(hr), hr ? hr->stride(0) : 0, ptr(w), p.codes, p.c_ld, p.scales,
                  p.s_ld, rs.data_ptr<float>(), ptr(dx), d, ptr(y), d, ptr(dw), ptr(ws), bytes, on.stream));
  return {dx, dw, y};
}

// -- rotary positions ------------------------------------------------------------------------------------------
// Whether no two elements of t share memory, by its strides.
bool separate(const Tensor& t) {
  std::vector<std::pair<int64_t, int64_t>> dims;
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1) dims.emplace_back(t.stride(i), t.size(i));
  std::sort(dims.begin(), dims.end());
  int64_t extent = 1;
  for (auto& [stride, size] : dims) {
    if (stride < extent) return false;
    extent = stride * size;
  }
  return true;
}

// Whether a and b, of one element size, have a byte in common; true too where that cannot be told in a few thousand steps.
// Elements at a + sum i_d s_d and b + sum j_d t_d meet where a bounded sum of the strides is the distance: one stride
// after another from the largest, each multiple from which the rest can still make up what is left.
bool overlap(const Tensor& a, const Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  const auto extent = [](const Tensor& t) {
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += t.stride(i) * (t.size(i) - 1);
    return (last + 1) * (int64_t)t.element_size();
  };
  const int64_t size = (int64_t)a.element_size();
  const int64_t bytes = reinterpret_cast<intptr_t>(b.data_ptr()) - reinterpret_cast<intptr_t>(a.data_ptr());
  if (bytes >= extent(a) || -bytes >= extent(b)) return false;
  if (bytes % size) return true;
  struct Term {
    int64_t stride, lo, hi;  // any multiple from lo to hi
  };
  std::vector<Term> terms;
  const auto add = [&](const Tensor& t, int64_t sign) {
    for (int64_t i = 0; i < t.dim(); ++i) {
      const int64_t stride = t.stride(i), last = t.size(i) - 1;
      if (stride == 0 || last == 0) continue;
      auto at = std::find_if(terms.begin(), terms.end(), [&](const Term& m) { return m.stride == stride; });
      if (at == terms.end()) at = terms.insert(at, {stride, 0, 0});
      (sign > 0 ? at->hi : at->lo) += sign * last;
    }
  };
  add(a, 1);
  add(b, -1);
  std::sort(terms.begin(), terms.end(), [](const Term& x, const Term& y) { return x.stride > y.stride; });
  const size_t n = terms.size();
  std::vector<int64_t> least(n + 1, 0), most(n + 1, 0), unit(n + 1, 0);  // what the terms from i on can make up; their divisor
  for (size_t i = n; i-- > 0;) {
    least[i] = least[i + 1] + terms[i].lo * terms[i].stride;
    most[i] = most[i + 1] + terms[i].hi * terms[i].stride;
    unit[i] = std::gcd(unit[i + 1], terms[i].stride);
  }
  const auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y < 0); };
  int steps = 1 << 14;
  const std::function<bool(size_t, int64_t)> meet = [&](size_t i, int64_t left) {
    if (i == n) return left == 0;
    if (left % unit[i]) return false;
    const int64_t s = terms[i].stride;
    const int64_t lo = std::max(terms[i].lo, -floor_div(most[i + 1] - left, s)), hi = std::min(terms[i].hi, floor_div(left - least[i + 1], s));
    for (int64_t c = lo; c <= hi; ++c)
      if (--steps < 0 || meet(i + 1, left - c * s)) return true;
    return false;
  };
  return meet(0, bytes / size);
}

// The same elements in the same places.
bool same_place(const Tensor& a, const Tensor& b) {
  if (a.data_ptr() != b.data_ptr()) return false;
  for (int64_t i = 0; i < a.dim(); ++i)
    if (a.size(i) > 1 && a.stride(i) != b.stride(i)) return false;
  return true;
}

gsa_rotary_side side_of(const Tensor& x, const Tensor& out) {
  return {ptr(x), ptr(out), (int32_t)x.size(2), x.stride(0), x.stride(1), x.stride(2), out.stride(0), out.stride(1),
          out.stride(2)};
}

struct Angles {
  optional<Tensor> inv_freq;  // fp64, contiguous
  optional<Tensor> cos, sin;
  int64_t rd = 0;
  double factor = 1;
  bool interleaved = false, inverse = false;
};

// q and k (of one shape but for the heads, as rotary checks them and autograd its gradients) into outputs like them.
void rotary_call(const Tensor& q_in, const optional<Tensor>& k_in, const Tensor& q_out, const optional<Tensor>& k_out,
                 const Tensor& positions, const Angles& a) {
  const On on(q_in);
  const Tensor q = q_in.stride(3) == 1 ? q_in : q_in.contiguous();
  optional<Tensor> k = k_in;
  if (k && k->stride(3) != 1) k = k->contiguous();
  const gsa_rotary_side sq = side_of(q, q_out), sk = k ? side_of(*k, *k_out) : gsa_rotary_side{};
  ok("gsa_rotary",
     api.rotary(code_of(q.scalar_type()), q.size(0), q.size(1), (int32_t)q.size(3), (int32_t)a.rd, &sq, k ? &sk : nullptr,
                positions.data_ptr<int64_t>(), positions.size(0) > 1 ? positions.stride(0) : 0, positions.stride(1),
                a.inv_freq ? a.inv_freq->data_ptr<double>() : nullptr, ptr(a.cos), ptr(a.sin),
                a.cos ? code_of(a.cos->scalar_type()) : 0, a.cos ? a.cos->stride(0) : 0, a.cos ? a.cos->size(0) : 0,
                (float)a.factor, a.interleaved, a.inverse, on.stream));
}

// [B or 1, L] int64.
Tensor whole_positions(const Tensor& given, int64_t B, int64_t L) {
  Tensor p = given.dim() == 1 ? given.unsqueeze(0) : given;
  TORCH_CHECK_VALUE(p.dim() == 2 && p.size(1) == L && (p.size(0) == 1 || p.size(0) == B), "positions ", given.sizes(), " for ", B,
                    " sequences of ", L, " tokens");
  TORCH_CHECK_VALUE(at::isIntegralType(p.scalar_type(), /*includeBool=*/false), "positions are integers");
  return p.scalar_type() == at::kLong ? p : p.to(at::kLong);
}

// The checks that need no positions; angles made whole.
void rotary_check(const Tensor& q, const optional<Tensor>& k, const Tensor& positions, Angles& a) {
  on_gpu(q);
  no_tangent(q);
  no_tangent(k);
  no_tangent(a.inv_freq);
  alike(k, q);
  beside(positions, q);
  code_of(q.scalar_type());
  TORCH_CHECK_VALUE(q.dim() == 4 && (!k || (k->dim() == 4 && k->size(0) == q.size(0) && k->size(1) == q.size(1) &&
                                            k->size(3) == q.size(3))),
                    "rotary takes q [B, L, H, D] and k [B, L, Hk, D], got q ", q.sizes());
  const int64_t D = q.size(3), heads = q.size(2) + (k ? k->size(2) : 0);
  if (a.cos) {
    TORCH_CHECK_VALUE(a.sin && a.cos->dim() == 2 && a.cos->sizes() == a.sin->sizes() && a.cos->strides() == a.sin->strides() &&
                          a.cos->stride(1) == 1 && a.cos->scalar_type() == a.sin->scalar_type() &&
                          a.cos->size(1) >= a.rd / 2,
                      "rotary tables are two [rows, >= rotary_dim/2] tensors of the same strides");
    beside(*a.cos, q);
    beside(*a.sin, q);
    code_of(a.cos->scalar_type());
  } else {
    TORCH_CHECK_VALUE(a.inv_freq && a.inv_freq->dim() == 1, "rotary takes inv_freq [rotary_dim/2]");
    beside(*a.inv_freq, q);
    a.rd = 2 * a.inv_freq->size(0);
    if (a.inv_freq->scalar_type() != at::kDouble || !a.inv_freq->is_contiguous())
      a.inv_freq = a.inv_freq->to(at::kDouble).contiguous();
  }
  TORCH_CHECK_VALUE(a.rd >= 2 && a.rd <= D && a.rd % 2 == 0 && D <= 1024 && heads <= 1024, "rotary: rotary_dim ", a.rd,
                    " of head dim ", D, ", at most 1024 wide and 1024 heads");
  const bool empty = q.numel() == 0 && (!k || k->numel() == 0);
  TORCH_CHECK_VALUE(empty || (q.size(2) > 0 && (!k || k->size(2) > 0)), "rotary: a tensor without heads");
}

using Pair = std::tuple<Tensor, optional<Tensor>>;

Pair rotary(const Tensor& q, const optional<Tensor>& k, const Tensor& positions, const optional<Tensor>& inv_freq,
            double factor, bool interleaved, bool inverse, const optional<Pair>& out,
            const optional<std::tuple<Tensor, Tensor>>& tables, int64_t rotary_dim) {
  Angles a;
  a.inv_freq = inv_freq;
  if (tables) std::tie(a.cos, a.sin) = *tables;
  a.rd = rotary_dim;
  a.factor = factor;
  a.interleaved = interleaved;
  a.inverse = inverse;
  rotary_check(q, k, positions, a);
  const Tensor pos = whole_positions(positions, q.size(0), q.size(1));
  Tensor q_out;
  optional<Tensor> k_out;
  if (out) {
    std::tie(q_out, k_out) = *out;
    TORCH_CHECK_VALUE(k.has_value() == k_out.has_value(), "rotary: an out tensor for each of q and k");
    for (int i = 0; i < (k ? 2 : 1); ++i) {
      const Tensor &x = i ? *k : q, &o = i ? *k_out : q_out;
      alike(o, x);
      no_tangent(o);
      overwritable(o);
      TORCH_CHECK_VALUE(o.sizes() == x.sizes() && (o.size(3) <= 1 || o.stride(3) == 1) && (o.is_contiguous() || separate(o)),
                        "rotary: out tensors have their inputs' shape, contiguous values and no two elements in one place");
    }
    // the kernel reads an input (unless it is laid out anew first) while others of its CTAs write; an output that is its input
    // itself is read and written by the same threads
    for (int i = 0; i < (k ? 2 : 1); ++i)
      for (int j = 0; j < (k ? 2 : 1); ++j) {
        const Tensor &o = i ? *k_out : q_out, &x = j ? *k : q;
        TORCH_CHECK_VALUE(x.stride(3) != 1 || (i == j && same_place(o, x)) || !overlap(o, x),
                          "rotary: an out tensor overlaps an input without being that input's own place");
      }
    TORCH_CHECK_VALUE(!k || !overlap(q_out, *k_out), "rotary: the out tensors overlap");
  } else {
    q_out = fresh(q);
    if (k) k_out = fresh(*k);
  }
  if (q.numel() == 0 && (!k || k->numel() == 0)) return {q_out, k_out};
  rotary_call(q, k, q_out, k_out, pos, a);
  if (out) {
    written(q_out);
    if (k_out) written(*k_out);
  }
  return {q_out, k_out};
}

void no_second_derivatives() {
  TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled(), "second derivatives of the training-step operators are not implemented");
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

optional<Tensor> given(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : std::nullopt; }

struct RotaryFn : torch::autograd::Function<RotaryFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const optional<Tensor>& k, const Tensor& positions,
                               const Tensor& inv_freq, double factor, bool interleaved) {
    Angles a;
    a.inv_freq = inv_freq;
    a.factor = factor;
    a.interleaved = interleaved;
    rotary_check(q, k, positions, a);
    const Tensor pos = whole_positions(positions, q.size(0), q.size(1));
    Tensor q_out = fresh(q);
    optional<Tensor> k_out;
    if (k) k_out = fresh(*k);
    if (q.numel() || (k && k->numel())) rotary_call(q, k, q_out, k_out, pos, a);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({pos, *a.inv_freq});
    ctx->saved_data["factor"] = factor;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["need_q"] = q.requires_grad();
    ctx->saved_data["need_k"] = k && k->requires_grad();
    if (k) return {q_out, *k_out};
    return {q_out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_derivatives();
    const auto saved = ctx->get_saved_variables();
    Angles a;
    a.inv_freq = saved[1];
    a.rd = 2 * saved[1].size(0);
    a.factor = ctx->saved_data["factor"].toDouble();
    a.interleaved = ctx->saved_data["interleaved"].toBool();
    a.inverse = true;
    Tensor in[2], out[2];
    if (ctx->saved_data["need_q"].toBool()) in[0] = grads[0];
    if (ctx->saved_data["need_k"].toBool()) in[1] = grads[1];
    for (int i = 0; i < 2; ++i)
      if (in[i].defined()) out[i] = fresh(in[i]);
    const int first = in[0].defined() ? 0 : 1;
    if (in[first].defined() && in[first].numel()) {
      const bool both = first == 0 && in[1].defined();
      rotary_call(in[first], both ? given(in[1]) : std::nullopt, out[first], both ? given(out[1]) : std::nullopt, saved[0],
                  a);
    }
    return {out[0], out[1], Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Pair rotary_autograd(const Tensor& q, const optional<Tensor>& k, const Tensor& positions, const Tensor& inv_freq, double factor,
                     bool interleaved) {
  const auto r = RotaryFn::apply(q, k, positions, inv_freq, factor, interleaved);
  return {r[0], k ? optional<Tensor>(r[1]) : std::nullopt};
}

struct SiluMulFn : torch::autograd::Function<SiluMulFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& gu) {
    auto [z, data] = silu_mul_packed(gu);
    ctx->save_for_backward({data});
    return z;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_derivatives();
    return {std::get<0>(silu_mul_packed_backward(grads[0], ctx->get_saved_variables()[0], false))};
  }
};

struct AddRMSNormFn : torch::autograd::Function<AddRMSNormFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& a, const Tensor& weight, double eps) {
    auto [h, y, data, rstd] = add_rmsnorm_packed(x, a, weight, eps);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({data, rstd, weight});
    ctx->saved_data["need_x"] = x.requires_grad();
    ctx->saved_data["need_a"] = a && a->requires_grad();
    ctx->saved_data["need_w"] = weight.requires_grad();
    if (h) return {y, *h};
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_derivatives();
    const auto saved = ctx->get_saved_variables();
    const Tensor dy = grads[0], dh = grads.size() > 1 ? grads[1] : Tensor();
    Tensor dx = dh, dw;
    if (dy.defined()) {
      auto r = rmsnorm_packed_backward(dy, saved[0], saved[1], saved[2], given(dh), false,
                                       ctx->saved_data["need_w"].toBool());
      dx = std::get<0>(r);
      if (std::get<1>(r)) dw = *std::get<1>(r);
    }
    return {ctx->saved_data["need_x"].toBool() ? dx : Tensor(), ctx->saved_data["need_a"].toBool() ? dx : Tensor(), dw,
            Tensor()};
  }
};

std::tuple<optional<Tensor>, Tensor> add_rmsnorm_autograd(const Tensor& x, const optional<Tensor>& a, const Tensor& weight,
                                                          double eps) {
  const auto r = AddRMSNormFn::apply(x, a, weight, eps);
  return {a ? optional<Tensor>(r[1]) : std::nullopt, r[0]};
}

// -- the loss --------------------------------------------------------------------------------------------------
std::tuple<Tensor, optional<Tensor>> next_token_loss(const Tensor& logits, const Tensor& labels_in, int64_t ignore_index,
                                                     bool want_grad) {
  on_gpu(logits);
  no_tangent(logits);
  TORCH_CHECK_VALUE(logits.dim() == 3 && logits.size(2) > 0 && labels_in.dim() == 2 && labels_in.size(0) == logits.size(0) &&
                        labels_in.size(1) == logits.size(1),
                    "next_token_loss takes logits [B, L, V] and labels [B, L], got ", logits.sizes(), " and ",
                    labels_in.sizes());
  beside(labels_in, logits);
  TORCH_CHECK_VALUE(at::isIntegralType(labels_in.scalar_type(), /*includeBool=*/false), "labels are integers");
  const int code = code_of(logits.scalar_type());
  const On on(logits);
  const Tensor labels = labels_in.scalar_type() == at::kLong ? labels_in : labels_in.to(at::kLong);
  const int64_t B = logits.size(0), L = logits.size(1), V = logits.size(2);
  const Tensor x = V == 1 || logits.stride(2) == 1 ? logits : logits.contiguous();
  Tensor loss = at::empty({}, logits.options().dtype(at::kFloat));
  const int64_t bytes = api.loss_ws();
  Tensor ws = at::empty({bytes}, logits.options().dtype(at::kByte));
  optional<Tensor> grad;
  if (want_grad) grad = fresh(logits);
  ok("gsa_next_token_loss",
     api.loss(code, B, L, V, ptr(x), x.stride(0), x.stride(1), labels.data_ptr<int64_t>(), labels.stride(0), labels.stride(1),
              ignore_index, loss.data_ptr<float>(), ptr(grad), L * V, V, ptr(ws), bytes, on.stream));
  return {loss, grad};
}

void scale_(const Tensor& x, const Tensor& factor) {
  on_gpu(x);
  no_tangent(x);
  no_tangent(factor);
  overwritable(x);
  beside(factor, x);
  TORCH_CHECK_VALUE(x.is_contiguous() && factor.numel() == 1 && factor.scalar_type() == at::kFloat,
                    "scale_ takes a contiguous tensor and a one-element fp32 factor");
  const On on(x);
  ok("gsa_scale", api.scale(code_of(x.scalar_type()), x.numel(), ptr(x), factor.data_ptr<float>(), on.stream));
  written(x);
}

struct LossFn : torch::autograd::Function<LossFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& labels, int64_t ignore_index) {
    auto [loss, grad] = next_token_loss(logits, labels, ignore_index, true);
    ctx->saved_data["grad"] = *grad;  // neither an input nor an output: held here until it is handed out
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_derivatives();
    const auto held = ctx->saved_data.find("grad");
    TORCH_CHECK(held != ctx->saved_data.end(), "fused_next_token_loss: its gradient was handed out by an earlier backward pass; call "
                                               "it again for another");
    const Tensor grad = held->second.toTensor();
    ctx->saved_data.erase(held);
    scale_(grad, grads[0]);
    return {grad, Tensor(), Tensor()};
  }
};

Tensor loss_autograd(const Tensor& logits, const Tensor& labels, int64_t ignore_index) {
  return LossFn::apply(logits, labels, ignore_index);
}

py::object* status_error = nullptr;  // gsa_b200._lib.GSAError

template <typename F>
void take(F& f, const py::dict& entries, const char* name) {
  f = reinterpret_cast<F>(entries[name].cast<uintptr_t>());
}

}  // namespace

PYBIND11_MODULE(_native, m) {
  m.def("bind", [](const py::dict& e, py::object error) {
    take(api.rotary, e, "gsa_rotary");
    take(api.pack, e, "gsa_pack_e4m3");
    take(api.unpack, e, "gsa_unpack_e4m3");
    take(api.silu_mul_pack, e, "gsa_silu_mul_pack");
    take(api.silu_mul_bwd, e, "gsa_silu_mul_packed_backward");
    take(api.norm_pack, e, "gsa_add_rmsnorm_pack");
    take(api.norm_ws, e, "gsa_rmsnorm_packed_workspace_size");
    take(api.norm_bwd, e, "gsa_rmsnorm_packed_backward");
    take(api.loss, e, "gsa_next_token_loss");
    take(api.loss_ws, e, "gsa_next_token_loss_workspace_size");
    take(api.scale, e, "gsa_scale");
    if (!status_error) status_error = new py::object(std::move(error));  // kept as long as the process lives
  });
  py::register_local_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Status& s) {
      PyErr_SetObject(status_error->ptr(), py::make_tuple(s.fn, s.status).ptr());
    } catch (const c10::ValueError& s) {
      PyErr_SetString(PyExc_ValueError, s.what_without_backtrace());
    } catch (const c10::NotImplementedError& s) {
      PyErr_SetString(PyExc_NotImplementedError, s.what_without_backtrace());
    }
  });
  // calls run without the interpreter lock, as torch's own do
  using free = py::call_guard<py::gil_scoped_release>;
  m.def("pack", &pack, free());
  m.def("unpack", &unpack, free());
  m.def("silu_mul_packed", &silu_mul_packed, free());
  m.def("silu_mul_packed_backward", &silu_mul_packed_backward, free());
  m.def("add_rmsnorm_packed", &add_rmsnorm_packed, free());
  m.def("rmsnorm_packed_backward", &rmsnorm_packed_backward, free());
  m.def("rotary", &rotary, free());
  m.def("overlap", &overlap, free());
  m.def("next_token_loss", &next_token_loss, free());
  m.def("scale_", &scale_, free());
  m.def("rotary_autograd", &rotary_autograd, free());
  m.def("silu_mul_autograd", [](const Tensor& gu) { return SiluMulFn::apply(gu); }, free());
  m.def("add_rmsnorm_autograd", &add_rmsnorm_autograd, free());
  m.def("loss_autograd", &loss_autograd, free());
}
