// pybind11 bindings of the 8-bit rows and products and of the gradient norm.
//
// Every entry checks its arguments before it asks where the tensors live, so
// that a wrong call is refused alike with and without a GPU (ops/reference.py
// refuses the same types, shapes, outputs and gradients); wrong values are
// ValueErrors.  Kernels run on the current stream of the tensors' own device,
// workspaces come from the caching allocator (and so belong to the graph, where
// one is being captured), and no call waits for the GPU.
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>
#include <utility>
#include <vector>

#include "grad_clip.h"
#include "int8.h"

extern "C" {
bool des_launch_quantize_rows(const void*, int, int64_t, int64_t, int8_t*,
                              int64_t, int64_t, float*, int64_t, int64_t, int,
                              hipStream_t);
bool des_launch_int8_product(const DesInt8Product*, hipStream_t);
void des_launch_pack_rows(const int8_t*, int64_t, int64_t, int8_t*, int64_t,
                          int64_t, int, hipStream_t);
void des_launch_square_sums(const DesClipTable*, int64_t, double*,
                            hipStream_t);
void des_launch_norm(const double*, int, float*, hipStream_t);
void des_launch_clip_scale(const DesClipTable*, int64_t, const double*, int,
                           double, float*, bool, bool, hipStream_t);
void des_launch_clip_small(const DesClipTable*, int64_t, double, float*, bool,
                           hipStream_t);
}

namespace {

using at::Tensor;
using c10::optional;

constexpr int64_t MAX_COLS = 131072;  // int32 sums of 127 * 127 stay in range
constexpr int64_t MAX_INT = 2147483647;
constexpr int64_t MAX_ROWS = 1 << 30;  // of a product: 32 bits hold a tile more

inline hipStream_t cur_stream() {
  return at::hip::getCurrentHIPStream().stream();
}

#define CHECK_LAUNCH() C10_HIP_CHECK(hipGetLastError())

int elem_of(at::ScalarType t, const char* what) {
  if (t == at::kFloat) return 0;
  if (t == at::kBFloat16) return 1;
  if (t == at::kHalf) return 2;
  TORCH_CHECK_VALUE(false, what, " must be float32, bfloat16 or float16, not ",
                    t);
}

// A tangent of forward mode would be lost as well, also where gradients are off.
void check_no_grad(const Tensor& t, const char* what) {
  TORCH_CHECK_VALUE(!(t.requires_grad() && at::GradMode::is_enabled()), what,
                    " requires a gradient, and this operator has none");
  TORCH_CHECK_VALUE(!t._fw_grad(0).defined(), what,
                    " carries a forward-mode gradient, and this operator has "
                    "none");
}

void check_place(const Tensor& t, const Tensor& like, const char* what) {
  TORCH_CHECK_VALUE(t.device() == like.device(), what, " is on ", t.device(),
                    ", other arguments are on ", like.device());
}

// Counts a write that autograd does not see by itself: a graph that saved the
// tensor then refuses to use it, instead of giving a wrong gradient.
void mark_written(const Tensor& t) { t.unsafeGetTensorImpl()->bump_version(); }

// Kernels read memory as it is: a view that torch negates when it reads it is
// written out first, and none is written to.  (resolve_neg alone goes through
// torch's dispatcher where there is nothing to do, too.)
Tensor plain(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

void check_plain(const Tensor& t, const char* what) {
  TORCH_CHECK_VALUE(!t.is_neg(), what, " must not be a negated view");
}

void check_gpu(const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "the HIP kernels need tensors on a GPU, not on ",
              t.device());
}

// the bytes that a tensor spans
std::pair<uintptr_t, uintptr_t> span(const Tensor& t) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(t.data_ptr());
  if (t.numel() == 0) return {p, p};
  int64_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
  return {p, p + (last + 1) * t.element_size()};
}

bool overlap(const Tensor& a, const Tensor& b) {
  const auto x = span(a), y = span(b);
  return x.first < y.second && y.first < x.second && x.first < x.second &&
         y.first < y.second;
}

// [..., cols] as lead x rows rows, where two strides can say so
struct Rows {
  int64_t lead = 1, rows = 1, sl = 0, sr = 0;
};

bool as_rows(const Tensor& t, Rows* r) {
  const int64_t last = t.dim() - 1;
  for (int64_t d = 0; d < last; ++d)
    if (t.size(d) == 0) {  // no rows: any strides will do
      *r = Rows{1, 0, 0, 0};
      return true;
    }
  if (t.size(last) > 1 && t.stride(last) != 1) return false;
  int64_t size[2] = {1, 1}, step[2] = {0, 0};
  int used = 0;  // from the inside out
  for (int64_t d = last - 1; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (used && t.stride(d) == size[used - 1] * step[used - 1]) {
      size[used - 1] *= t.size(d);
    } else {
      if (used == 2) return false;
      size[used] = t.size(d);
      step[used] = t.stride(d);
      ++used;
    }
  }
  r->rows = size[0];
  r->sr = step[0];
  r->lead = size[1];
  r->sl = step[1];
  return true;
}

// whether rows of a tensor that is written are apart from one another
bool rows_apart(const Rows& r, int64_t cols) {
  int64_t in = r.sr, nin = r.rows, outer = r.sl, nout = r.lead;
  if (nin > 1 && nout > 1 && in > outer) {
    std::swap(in, outer);
    std::swap(nin, nout);
  }
  if (nin > 1 && in < cols) return false;
  const int64_t inner = nin > 1 ? in * (nin - 1) + cols : cols;
  return nout <= 1 || outer >= inner;
}

std::vector<int64_t> lead_shape(const Tensor& x) {
  return {x.sizes().begin(), x.sizes().end() - 1};
}

// Bytes from row to row of fresh codes: whole pieces of 16, which the products'
// wide loads like, or whole lines of 128, where that adds 1/16 at most (a product
// of 8192 x 512 x 3136 with rows of 3200 bytes: in tiles of 64 x 64 21.6 us instead
// of 24.8, of 128 x 64 20.3 instead of 21.4, of 128 x 128 no difference).
int64_t row_step(int64_t cols) {
  const int64_t line = (cols + 127) / 128 * 128;
  return line - cols <= cols / 16 ? line : (cols + 15) / 16 * 16;
}

// codes for rows of x's shape; the last row's gap belongs to the storage
Tensor new_codes(const Tensor& x) {
  const auto shape = x.sizes();
  std::vector<int64_t> strides(shape.size(), 1);
  int64_t total = row_step(shape.back());
  for (int64_t d = (int64_t)shape.size() - 2; d >= 0; --d) {
    strides[d] = total;
    total *= std::max<int64_t>(1, shape[d]);
  }
  Tensor q = at::empty({total}, x.options().dtype(at::kChar));
  q.unsafeGetTensorImpl()->set_sizes_and_strides(shape, strides);
  return q;
}

void check_float_rows(const Tensor& x) {
  elem_of(x.scalar_type(), "x");
  TORCH_CHECK_VALUE(x.dim() >= 1, "x must have at least one dimension");
  TORCH_CHECK_VALUE(x.size(-1) <= MAX_COLS, "rows of at most ", MAX_COLS,
                    " values, not ", x.size(-1));
  check_no_grad(x, "x");
}

void launch_quantize(const Tensor& x, const Tensor& q, const Tensor& s) {
  Rows xr, qr;
  TORCH_INTERNAL_ASSERT(as_rows(x, &xr) && as_rows(q, &qr));
  const int64_t cols = x.size(-1);
  const int64_t rows = xr.lead * xr.rows;
  if (rows == 0) return;
  if (qr.lead != xr.lead || qr.rows != xr.rows) {
    // the two tensors' rows come in other groups: both by the finer grouping
    if (xr.lead == 1 && qr.rows > 0) {
      xr = Rows{qr.lead, qr.rows, qr.rows * xr.sr, xr.sr};
    } else {
      TORCH_INTERNAL_ASSERT(qr.lead == 1);
      qr = Rows{xr.lead, xr.rows, xr.rows * qr.sr, qr.sr};
    }
  }
  TORCH_CHECK_VALUE(
      rows <= MAX_INT &&
          des_launch_quantize_rows(
              x.data_ptr(), elem_of(x.scalar_type(), "x"), xr.sl, xr.sr,
              q.data_ptr<int8_t>(), qr.sl, qr.sr, s.data_ptr<float>(), xr.lead,
              xr.rows, (int)cols, cur_stream()),
      rows, " rows are too many for one call");
  CHECK_LAUNCH();
}

// x by two strides and a unit step, copied where it has other strides.  Without
// elements any strides count as contiguous, and a copy would keep them.
Tensor row_view(const Tensor& x) {
  if (x.numel() == 0) return at::empty(x.sizes(), x.options());
  Rows r;
  return as_rows(x, &r) ? x : x.contiguous();
}

std::pair<Tensor, Tensor> quantize_rows(const Tensor& x_,
                                        const optional<Tensor>& q_,
                                        const optional<Tensor>& s_) {
  check_float_rows(x_);
  TORCH_CHECK_VALUE(q_.has_value() == s_.has_value(),
                    "out holds codes and scales, or is None");
  const auto shape = lead_shape(x_);
  if (q_.has_value()) {
    Rows r;
    TORCH_CHECK_VALUE(q_->scalar_type() == at::kChar && q_->sizes() == x_.sizes(),
                      "out[0] must be int8 of x's shape");
    TORCH_CHECK_VALUE(s_->scalar_type() == at::kFloat &&
                          s_->sizes() == at::IntArrayRef(shape) &&
                          s_->is_contiguous(),
                      "out[1] must be contiguous float32 of x's shape without "
                      "its last dimension");
    check_place(*q_, x_, "out[0]");
    check_place(*s_, x_, "out[1]");
    check_plain(*q_, "out[0]");
    check_plain(*s_, "out[1]");
    check_no_grad(*s_, "out[1]");
    TORCH_CHECK_VALUE(as_rows(*q_, &r) && rows_apart(r, x_.size(-1)),
                      "out[0] must hold its rows apart, by two strides and "
                      "with a last stride of 1");
    TORCH_CHECK_VALUE(!overlap(*q_, x_) && !overlap(*s_, x_) &&
                          !overlap(*q_, *s_),
                      "out overlaps x or itself");
  }
  check_gpu(x_);
  const c10::DeviceGuard guard(x_.device());
  Tensor q = q_.has_value() ? *q_ : new_codes(x_);
  Tensor s = s_.has_value() ? *s_
                            : at::empty(shape, x_.options().dtype(at::kFloat));
  Tensor x = row_view(plain(x_));
  Rows xr, qr;
  as_rows(x, &xr);
  as_rows(q, &qr);
  if (xr.lead != 1 && qr.lead != 1 && (xr.lead != qr.lead || xr.rows != qr.rows))
    x = x.contiguous();  // rows grouped unlike those of out
  if (q_.has_value()) {
    mark_written(q);
    mark_written(s);
  }
  launch_quantize(x, q, s);
  return {q, s};
}

int act_of(const std::string& name) {
  if (name == "none") return 0;
  if (name == "relu") return 1;
  if (name == "tanh") return 2;
  TORCH_CHECK_VALUE(false, "activation must be none, relu or tanh, not ", name);
}

// what both products check of their weights and results; x gives only shapes
std::vector<int64_t> check_product(const Tensor& x, const Tensor& wq,
                                   const Tensor& sw,
                                   const optional<Tensor>& bias,
                                   at::ScalarType out_dtype,
                                   const optional<Tensor>& out) {
  TORCH_CHECK_VALUE(wq.scalar_type() == at::kChar, "wq must be int8, not ",
                    wq.scalar_type());
  TORCH_CHECK_VALUE(wq.dim() == 2 || wq.dim() == 3,
                    "wq must be [channels, cols] or [members, channels, cols]");
  TORCH_CHECK_VALUE(wq.dim() == 2 || x.dim() == 3,
                    "members' weights need x of [members, tokens, cols]");
  TORCH_CHECK_VALUE(x.size(-1) == wq.size(-1), "rows of ", x.size(-1),
                    " values against weights of ", wq.size(-1));
  TORCH_CHECK_VALUE(wq.dim() == 2 || x.size(0) == wq.size(0), "x has ",
                    x.size(0), " members, the weights ", wq.size(0));
  TORCH_CHECK_VALUE(x.size(-1) <= MAX_COLS, "rows of at most ", MAX_COLS,
                    " values, not ", x.size(-1));
  const auto channels = lead_shape(wq);
  TORCH_CHECK_VALUE(sw.scalar_type() == at::kFloat &&
                        sw.sizes() == at::IntArrayRef(channels),
                    "sw must be float32 of wq's shape without its last "
                    "dimension");
  check_place(wq, x, "wq");
  check_place(sw, x, "sw");
  check_no_grad(sw, "sw");
  if (bias.has_value()) {
    TORCH_CHECK_VALUE(bias->scalar_type() == at::kFloat &&
                          bias->sizes() == sw.sizes(),
                      "bias must be float32 of sw's shape");
    check_place(*bias, x, "bias");
    check_no_grad(*bias, "bias");
  }
  elem_of(out_dtype, "out_dtype");
  auto shape = lead_shape(x);
  shape.push_back(wq.size(-2));
  if (out.has_value()) {
    TORCH_CHECK_VALUE(out->scalar_type() == out_dtype &&
                          out->sizes() == at::IntArrayRef(shape) &&
                          out->is_contiguous(),
                      "out must be contiguous, of out_dtype and of shape ",
                      at::IntArrayRef(shape));
    check_place(*out, x, "out");
    check_no_grad(*out, "out");
    check_plain(*out, "out");
    TORCH_CHECK_VALUE(!overlap(*out, x) && !overlap(*out, wq) &&
                          !overlap(*out, sw) &&
                          !(bias.has_value() && overlap(*out, *bias)),
                      "out overlaps an argument");
  }
  return shape;
}

// whether every row's last 16 codes lie inside the tensor's storage
bool whole_rows(const Tensor& t) {
  int64_t last = t.storage_offset();
  for (int64_t d = 0; d + 1 < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
  return last + (t.size(-1) + 15) / 16 * 16 <= (int64_t)t.storage().nbytes();
}

// The tiled kernel reads whole pieces of 16 codes at addresses of 16: rows that
// lie otherwise are copied.  `kept` holds the copy until the product is
// launched.
const int8_t* aligned_rows(const int8_t* rows, int64_t* sb, int64_t* sr,
                           int64_t B, int64_t n, int64_t K, bool whole,
                           const Tensor& like, Tensor* kept) {
  const int64_t lead = B > 1 && *sb != 0 ? B : 1;
  if (whole && reinterpret_cast<uintptr_t>(rows) % 16 == 0 &&
      (n == 1 || *sr % 16 == 0) && (lead == 1 || *sb % 16 == 0))
    return rows;
  const int64_t step = (K + 15) / 16 * 16;
  *kept = at::empty({lead * n * step}, like.options().dtype(at::kChar));
  des_launch_pack_rows(rows, *sb, *sr, kept->data_ptr<int8_t>(), lead, n,
                       (int)K, cur_stream());
  CHECK_LAUNCH();
  *sr = step;
  *sb = lead == 1 ? 0 : n * step;
  return kept->data_ptr<int8_t>();
}

// x: codes with their scales sx, or (sx undefined) float rows
Tensor product(const Tensor& x_, const Tensor& sx_, const Tensor& wq_,
               const Tensor& sw_, const optional<Tensor>& bias_, int act,
               at::ScalarType out_dtype, const optional<Tensor>& out,
               const std::vector<int64_t>& shape) {
  Tensor y =
      out.has_value() ? *out : at::empty(shape, sw_.options().dtype(out_dtype));
  if (out.has_value()) mark_written(y);
  if (y.numel() == 0) return y;
  DesInt8Product p = {};
  const bool members = wq_.dim() == 3;
  Tensor x = row_view(plain(x_));
  if (!members) {
    Rows r;
    as_rows(x, &r);
    if (r.lead != 1) x = x.contiguous();
    as_rows(x, &r);
    TORCH_CHECK_VALUE(r.rows <= MAX_ROWS, "too many rows: ", r.rows);
    p.B = 1;
    p.M = (int32_t)r.rows;
    p.xsb = 0;
    p.xsr = r.sr;
  } else {
    TORCH_CHECK_VALUE(x.size(1) <= MAX_ROWS, "too many rows: ", x.size(1));
    p.B = x.size(0);
    p.M = (int32_t)x.size(1);
    p.xsb = x.stride(0);
    p.xsr = x.stride(1);
  }
  const int64_t K = x.size(-1);
  Tensor sx;
  if (sx_.defined()) {
    sx = plain(sx_).contiguous();
  } else if (!des_int8_fused(p.M, K)) {
    const Tensor q = new_codes(x);
    sx = at::empty(lead_shape(x), x.options().dtype(at::kFloat));
    launch_quantize(x, q, sx);
    x = q;
    p.xsr = members ? q.stride(1) : row_step(K);
    p.xsb = members ? q.stride(0) : 0;
  }
  if (sx.defined()) {
    p.x = x.data_ptr<int8_t>();
    p.sx = sx.data_ptr<float>();
    p.xwhole = whole_rows(x);
  } else {
    p.xf = x.data_ptr();
    p.xelem = elem_of(x.scalar_type(), "x");
  }
  Tensor wq = plain(wq_);
  if (K > 1 && wq.stride(-1) != 1) wq = wq.contiguous();
  TORCH_CHECK_VALUE(wq.size(-2) <= MAX_ROWS, "too many channels");
  p.N = (int32_t)wq.size(-2);
  p.K = (int32_t)K;
  p.wsb = members ? wq.stride(0) : 0;
  p.wsr = wq.stride(-2);
  p.wwhole = whole_rows(wq);
  const Tensor sw = plain(sw_).contiguous();
  const Tensor bias =
      bias_.has_value() ? plain(*bias_).contiguous() : Tensor();
  p.w = wq.data_ptr<int8_t>();
  p.sw = sw.data_ptr<float>();
  p.bias = bias.defined() ? bias.data_ptr<float>() : nullptr;
  p.y = y.data_ptr();
  p.act = act;
  p.out = elem_of(out_dtype, "out_dtype");
  Tensor x_copy, w_copy;
  if (K > 0 && des_int8_plan(p.B, p.M, p.N, p.K) == DES_INT8_TILED) {
    p.x = aligned_rows(p.x, &p.xsb, &p.xsr, p.B, p.M, K, p.xwhole, y, &x_copy);
    p.w = aligned_rows(p.w, &p.wsb, &p.wsr, p.B, p.N, K, p.wwhole, y, &w_copy);
  }
  TORCH_CHECK_VALUE(des_launch_int8_product(&p, cur_stream()), "a product of ",
                    p.B, " x ", p.M, " x ", p.N,
                    " results is too large for one call");
  CHECK_LAUNCH();
  return y;
}

Tensor int8_matmul(const Tensor& xq, const Tensor& sx, const Tensor& wq,
                   const Tensor& sw, const optional<Tensor>& bias,
                   const std::string& activation, at::ScalarType out_dtype,
                   const optional<Tensor>& out) {
  TORCH_CHECK_VALUE(xq.scalar_type() == at::kChar, "xq must be int8, not ",
                    xq.scalar_type());
  TORCH_CHECK_VALUE(xq.dim() >= 1, "xq must have at least one dimension");
  TORCH_CHECK_VALUE(sx.scalar_type() == at::kFloat &&
                        sx.sizes() == at::IntArrayRef(lead_shape(xq)),
                    "sx must be float32 of xq's shape without its last "
                    "dimension");
  check_place(sx, xq, "sx");
  check_no_grad(sx, "sx");
  const int act = act_of(activation);
  const auto shape = check_product(xq, wq, sw, bias, out_dtype, out);
  TORCH_CHECK_VALUE(!(out.has_value() && overlap(*out, sx)),
                    "out overlaps an argument");
  check_gpu(xq);
  const c10::DeviceGuard guard(xq.device());
  return product(xq, sx, wq, sw, bias, act, out_dtype, out, shape);
}

Tensor int8_linear(const Tensor& x_, const Tensor& wq, const Tensor& sw,
                   const optional<Tensor>& bias, const std::string& activation,
                   at::ScalarType out_dtype, const optional<Tensor>& out) {
  check_float_rows(x_);
  const int act = act_of(activation);
  const auto shape = check_product(x_, wq, sw, bias, out_dtype, out);
  check_gpu(x_);
  const c10::DeviceGuard guard(x_.device());
  return product(x_, Tensor(), wq, sw, bias, act, out_dtype, out, shape);
}

// ---------------------------------------------------------------------------

void check_tensors(const std::vector<Tensor>& tensors) {
  TORCH_CHECK_VALUE(!tensors.empty(), "no tensors");
  for (const Tensor& t : tensors) {
    elem_of(t.scalar_type(), "tensors");
    check_place(t, tensors[0], "a tensor");
    check_no_grad(t, "a tensor");
  }
}

int64_t total_of(const std::vector<Tensor>& tensors) {
  int64_t total = 0;
  for (const Tensor& t : tensors) total += t.numel();
  return total;
}

// Few values in few tensors: one block does it all in one launch.
bool is_small(const std::vector<Tensor>& tensors) {
  return tensors.size() <= DES_CLIP_TENSORS && total_of(tensors) <= 1 << 15;
}

// A share of a tensor is one block's work (a wave's, where it is small): 2^12
// values, or more where a single tensor of that size would give over 2048 blocks,
// since each block of the second pass joins all sums.  Every tensor takes a block
// at least, so a list of T tensors has up to 2048 + T of them, and joining the sums
// grows with the square of T: 10000 small tensors read 0.8 GB of sums from caches.
int64_t share_of(const std::vector<Tensor>& tensors) {
  if (is_small(tensors)) return 1 << 10;
  const int64_t total = total_of(tensors);
  int64_t share = 1 << 12;
  while (total / share > 2048) share *= 2;
  return share;
}

struct Tables {
  std::vector<DesClipTable> tables;
  int64_t blocks = 0;
};

Tables tables_of(const std::vector<Tensor>& in, const std::vector<Tensor>& out,
                 int64_t share) {
  Tables r;
  for (size_t i = 0; i < in.size(); ++i) {
    if (i % DES_CLIP_TENSORS == 0) {
      r.tables.emplace_back();
      r.tables.back().count = 0;
      r.tables.back().first[0] = 0;
    }
    DesClipTable& t = r.tables.back();
    const int at = t.count++;
    t.in[at] = in[i].data_ptr();
    t.out[at] = out.empty() ? nullptr : out[i].data_ptr();
    t.numel[at] = in[i].numel();
    t.elem[at] = (uint8_t)elem_of(in[i].scalar_type(), "tensors");
    const int64_t blocks =
        std::max<int64_t>(1, (in[i].numel() + share - 1) / share);
    t.first[at + 1] = t.first[at] + (int32_t)blocks;
    r.blocks += blocks;
  }
  return r;
}

Tensor square_sums(const Tables& tables, int64_t share, const Tensor& like) {
  Tensor sums = at::empty({tables.blocks}, like.options().dtype(at::kDouble));
  double* p = sums.data_ptr<double>();
  for (const DesClipTable& t : tables.tables) {
    des_launch_square_sums(&t, share, p, cur_stream());
    CHECK_LAUNCH();
    p += t.first[t.count];
  }
  return sums;
}

Tensor global_norm(const std::vector<Tensor>& tensors) {
  check_tensors(tensors);
  check_gpu(tensors[0]);
  const c10::DeviceGuard guard(tensors[0].device());
  std::vector<Tensor> in;
  for (const Tensor& t : tensors)
    in.push_back(plain(t).contiguous());
  const int64_t share = share_of(in);
  const Tables tables = tables_of(in, {}, share);
  Tensor norm = at::empty({}, in[0].options().dtype(at::kFloat));
  if (is_small(in)) {
    des_launch_clip_small(&tables.tables[0], share, 0.0,
                          norm.data_ptr<float>(), false, cur_stream());
    CHECK_LAUNCH();
    return norm;
  }
  const Tensor sums = square_sums(tables, share, in[0]);
  des_launch_norm(sums.data_ptr<double>(), (int)tables.blocks,
                  norm.data_ptr<float>(), cur_stream());
  CHECK_LAUNCH();
  return norm;
}

// -> (the clipped tensors, or None where they are `out`; the norm)
std::pair<optional<std::vector<Tensor>>, Tensor> clip_by_global_norm(
    const std::vector<Tensor>& tensors, double max_norm,
    const optional<std::vector<Tensor>>& out) {
  check_tensors(tensors);
  TORCH_CHECK_VALUE(max_norm >= 0, "max_norm must be at least 0, not ",
                    max_norm);
  if (out.has_value()) {
    TORCH_CHECK_VALUE(out->size() == tensors.size(), "out holds ", out->size(),
                      " tensors for ", tensors.size());
    // who reads and who writes which bytes: a write may meet no other write,
    // and no read but that of its own tensor, in place
    struct Use {
      uintptr_t begin, end;
      size_t of;
      bool write;
    };
    std::vector<Use> uses;
    for (size_t i = 0; i < tensors.size(); ++i) {
      const Tensor& o = (*out)[i];
      TORCH_CHECK_VALUE(o.scalar_type() == tensors[i].scalar_type() &&
                            o.sizes() == tensors[i].sizes() &&
                            o.is_contiguous(),
                        "out[", i, "] must be contiguous, of its tensor's type "
                        "and shape");
      check_place(o, tensors[0], "out");
      check_no_grad(o, "out");
      check_plain(o, "out");
      if (o.numel() == 0) continue;
      const auto a = span(tensors[i]), b = span(o);
      uses.push_back({b.first, b.second, i, true});
      if (a != b) uses.push_back({a.first, a.second, i, false});
    }
    std::sort(uses.begin(), uses.end(),
              [](const Use& a, const Use& b) { return a.begin < b.begin; });
    uintptr_t written = 0, read = 0;
    for (const Use& u : uses) {
      TORCH_CHECK_VALUE(u.begin >= written && (!u.write || u.begin >= read),
                        "out[", u.of, "] overlaps another tensor");
      (u.write ? written : read) = std::max(u.write ? written : read, u.end);
    }
  }
  check_gpu(tensors[0]);
  const c10::DeviceGuard guard(tensors[0].device());
  std::vector<Tensor> in, to;
  auto result = [&]() -> optional<std::vector<Tensor>> {
    if (out.has_value()) return c10::nullopt;
    return to;
  };
  for (size_t i = 0; i < tensors.size(); ++i) {
    if (out.has_value()) mark_written((*out)[i]);
    in.push_back(plain(tensors[i]).contiguous());
    to.push_back(out.has_value() ? (*out)[i] : at::empty_like(in[i]));
  }
  const int64_t share = share_of(in);
  const Tables tables = tables_of(in, to, share);
  Tensor norm = at::empty({}, in[0].options().dtype(at::kFloat));
  if (is_small(in)) {
    des_launch_clip_small(&tables.tables[0], share, max_norm,
                          norm.data_ptr<float>(), true, cur_stream());
    CHECK_LAUNCH();
    return {result(), norm};
  }
  const Tensor sums = square_sums(tables, share, in[0]);
  bool first = true;
  int64_t bytes = 0;
  for (const Tensor& t : in) bytes += t.nbytes();
  for (const DesClipTable& t : tables.tables) {
    des_launch_clip_scale(&t, share, sums.data_ptr<double>(),
                          (int)tables.blocks, max_norm,
                          norm.data_ptr<float>(), first, bytes > 32 << 20,
                          cur_stream());
    CHECK_LAUNCH();
    first = false;
  }
  return {result(), norm};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("quantize_rows", &quantize_rows, "float rows -> 8-bit rows and scales",
        py::arg("x"), py::arg("q") = py::none(), py::arg("s") = py::none());
  m.def("int8_matmul", &int8_matmul, "8-bit rows x 8-bit weights",
        py::arg("xq"), py::arg("sx"), py::arg("wq"), py::arg("sw"),
        py::arg("bias"), py::arg("activation"), py::arg("out_dtype"),
        py::arg("out"));
  m.def("int8_linear", &int8_linear, "float rows x 8-bit weights",
        py::arg("x"), py::arg("wq"), py::arg("sw"), py::arg("bias"),
        py::arg("activation"), py::arg("out_dtype"), py::arg("out"));
  m.def("global_norm", &global_norm, "norm over all tensors",
        py::arg("tensors"));
  m.def("clip_by_global_norm", &clip_by_global_norm,
        "tensors bounded by their global norm", py::arg("tensors"),
        py::arg("max_norm"), py::arg("out"));
}
