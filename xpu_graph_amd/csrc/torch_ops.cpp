// torch.ops.xpu_ops implementations in C++: query / key preparation and linear attention over the C entry points of
// xpu_graph_amd.h.  These ops are called once per layer and token, or once per layer on both sides of a training step, where the
// interpreter would cost more than the kernels (a call 13 to 30 us, its share of a backward pass twice that, since it runs on the
// autograd engine's thread).  Schemas and the shape-only Meta implementations are in ops.py; the checks here are the same.
//
// Each op: checks, operands that the kernels can read (a copy only where strides or alignment do not fit), results from the
// caching allocator, one call on the tensors' device and its current stream.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_strided.h>
#include <ATen/ops/zeros_like.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <algorithm>
#include <array>
#include <tuple>

#include "../../include/xpu_graph_amd.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kMaxAxes = 4, kMaxHeadDim = 512;
// Tokens further apart than this are copied together first: the chunked kernels address 32 rows by 32-bit offsets.
constexpr int64_t kMaxPitch = 1 << 26;

int code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return XG_F32;
    case at::kHalf: return XG_F16;
    case at::kBFloat16: return XG_BF16;
    default: TORCH_CHECK_TYPE(false, "xpu_ops: dtype ", t, " has no mi355x kernel");
  }
}

void check_status(int status, const char* what) {
  TORCH_CHECK(status == XG_OK, what, " failed: ", xg_status_string(status), " (status ", status, ")");
}

void* ptr(const Tensor& t) { return t.data_ptr(); }
void* ptr(const OptTensor& t) { return t.has_value() && t->defined() ? t->data_ptr() : nullptr; }
bool has(const OptTensor& t) { return t.has_value() && t->defined(); }
bool misaligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0; }

void same_device(const Tensor& first, std::initializer_list<const OptTensor*> others) {
  for (const OptTensor* t : others)
    TORCH_CHECK_VALUE(!has(*t) || (*t)->device() == first.device(), "xpu_ops: tensors on different devices (", first.device(), " and ", (*t)->device(), ")");
}

// Unit last stride, the others multiples of 16 bytes (dimensions of size 1 have none that counts).
bool readable(const Tensor& t) {
  const int64_t per16 = 16 / t.element_size(), n = t.dim();
  if (t.stride(n - 1) != 1) return false;
  for (int64_t i = 0; i + 1 < n; ++i)
    if (t.size(i) != 1 && t.stride(i) % per16) return false;
  return true;
}

// The strides are a permutation of a contiguous block.
bool dense(const Tensor& t) {
  std::array<std::pair<int64_t, int64_t>, 4> dims;
  int n = 0;
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) != 1) dims[n++] = {t.stride(i), t.size(i)};
  std::sort(dims.begin(), dims.begin() + n);
  int64_t expect = 1;
  for (int i = 0; i < n; ++i) {
    if (dims[i].first != expect) return false;
    expect *= dims[i].second;
  }
  return true;
}

// A result in the layout of `t` where that is dense and readable; where `t` is a part of something else, such as one of several
// projections side by side, dense with the dimensions in the order of its strides (rows of a token stay together: the kernels
// write 10 to 15 % faster than one head after the other); else contiguous.
Tensor result_like(const Tensor& t, int64_t max_pitch = INT64_MAX) {
  if (t.stride(3) == 1 && t.numel() > 0) {
    std::array<int64_t, 4> to{};
    if (readable(t) && dense(t)) {
      std::copy(t.strides().begin(), t.strides().end(), to.begin());
    } else {
      std::array<int, 3> order{0, 1, 2};
      std::stable_sort(order.begin(), order.end(), [&](int a, int b) { return t.stride(a) < t.stride(b); });
      int64_t next = t.size(3);
      bool spread = true;
      for (int i : order) {
        spread = spread && (t.size(i) == 1 || t.stride(i) > 0);
        to[i] = next;
        next *= t.size(i);
      }
      if (!spread) return at::empty(t.sizes(), t.options());
      to[3] = 1;
    }
    if (t.size(2) == 1 || to[2] < max_pitch) return at::empty_strided(t.sizes(), to, t.options());
  }
  return at::empty(t.sizes(), t.options());
}

// The tensor, or a copy that the kernels can read.
Tensor operand(const Tensor& t) {
  Tensor x = readable(t) ? t : t.contiguous();
  return misaligned(x) ? x.clone(at::MemoryFormat::Contiguous) : x;
}
Tensor token_operand(const Tensor& t) {
  Tensor x = operand(t);
  return x.size(2) == 1 || x.stride(2) < kMaxPitch ? x : x.contiguous();
}

// Strides as the entry points take them: 0 where a dimension has one element, whatever the tensor says there.
struct Strides {
  std::array<int64_t, 4> s{};
  operator const int64_t*() const { return s.data(); }
};
Strides strides(const Tensor& t) {
  Strides r;
  for (int64_t i = 0; i < 4; ++i) r.s[i] = t.size(i) == 1 ? 0 : t.stride(i);
  return r;
}

// Runs `launch(stream)` on the tensor's device, whatever the current one is.
template <typename F>
void launch(const Tensor& on, const char* what, F&& f) {
  const c10::DeviceGuard guard(on.device());
  check_status(f(c10::hip::getCurrentHIPStream(on.device().index()).stream()), what);
}

// ------------------------------------------------------------------- rotation
struct Rotary {
  xg_rotary r{};
  Tensor cos, sin;
  std::array<uint8_t, kMaxHeadDim / 2> pair_axis;

  Rotary(const Tensor& x, const Tensor& cos_in, const Tensor& sin_in, const OptTensor& positions, at::IntArrayRef sections, bool interleaved) {
    TORCH_CHECK_VALUE(x.dim() == 4, "rope_axes: q, k or x must be [B, H, S, D]");
    const int64_t B = x.size(0), S = x.size(2), D = x.size(3), axes = std::max<int64_t>(sections.size(), 1);
    TORCH_CHECK_VALUE(D > 0 && D % 16 == 0 && D <= kMaxHeadDim, "rope_axes: head dim must be a multiple of 16, at most ", kMaxHeadDim);
    bool flat = cos_in.sizes() == sin_in.sizes() && cos_in.dim() >= 1;
    for (int64_t i = 0; flat && i + 2 < cos_in.dim(); ++i) flat = cos_in.size(i) == 1;
    TORCH_CHECK_VALUE(flat, "rope_axes: cos / sin must be [P, R] or [P, R/2] tables of one shape (leading dims of size 1 allowed)");
    const auto table_type = cos_in.scalar_type();
    TORCH_CHECK_TYPE(table_type == sin_in.scalar_type() && (table_type == x.scalar_type() || table_type == at::kFloat),
                     "rope_axes: cos / sin must share a dtype, that of x or float32");
    TORCH_CHECK_VALUE(axes <= kMaxAxes, "rope_axes: at most ", kMaxAxes, " axes");
    int64_t pairs = sections.empty() ? D / 2 : 0;
    for (int64_t n : sections) {
      TORCH_CHECK_VALUE(n >= 0 && n <= D, "rope_axes: sections are the pairs of each axis");
      pairs += n;
    }
    const int64_t rot = 2 * pairs, cols = cos_in.size(-1), rows = cos_in.dim() > 1 ? cos_in.size(-2) : 1;
    TORCH_CHECK_VALUE(rot > 0 && rot <= D && rot % 16 == 0 && (cols == rot || cols == rot / 2),
                      "rope_axes: 2 * sum(sections) = R must be a multiple of 16 up to the head dim, the tables R or R/2 columns wide");
    same_device(x, {&positions});
    TORCH_CHECK_VALUE(cos_in.device() == x.device() && sin_in.device() == x.device(), "xpu_ops: tensors on different devices");
    if (!has(positions)) {
      TORCH_CHECK_VALUE(axes == 1 && (rows == S || rows == 1),
                        "rope_axes: without positions there is one axis and the tables have one row per token, or one row");
    } else {
      const Tensor& p = *positions;
      const int64_t n = p.dim();
      TORCH_CHECK_TYPE(p.scalar_type() == at::kInt || p.scalar_type() == at::kLong, "rope_axes: positions must be int32 or int64");
      TORCH_CHECK_VALUE((axes == 1 ? n >= 1 && n <= 3 : n == 3) && (n < 3 ? 1 : p.size(0)) == axes && (n < 2 || p.size(-2) == 1 || p.size(-2) == B) &&
                            p.size(-1) == S,
                        "rope_axes: positions must be [axes, B, S] ([S] or [B, S] with one axis; a batch dim of 1 is shared)");
      TORCH_CHECK_VALUE(rows > 0, "rope_axes: the tables are empty");
      r.positions = p.data_ptr();
      r.positions_64bit = p.scalar_type() == at::kLong;
      r.pos_strides[0] = n == 3 ? p.stride(0) : 0;
      r.pos_strides[1] = n >= 2 && p.size(-2) > 1 ? p.stride(-2) : 0;
      r.pos_strides[2] = p.stride(-1);
    }
    cos = cos_in;
    sin = sin_in;
    const int64_t per16 = 16 / cos.element_size();
    const bool in_place = cos.dim() > 1 && cos.strides() == sin.strides() && cos.stride(-1) == 1 && cos.stride(-2) >= cols &&
                          cos.stride(-2) % per16 == 0 && !misaligned(cos) && !misaligned(sin);
    if (!in_place) {
      cos = cos.reshape({rows, cols}).clone(at::MemoryFormat::Contiguous);
      sin = sin.reshape({rows, cols}).clone(at::MemoryFormat::Contiguous);
    }
    r.cos_table = cos.data_ptr();
    r.sin_table = sin.data_ptr();
    r.table_rows = rows;
    r.table_cols = cols;
    r.table_stride = cos.stride(-2) >= cols ? cos.stride(-2) : cols;
    r.rot_dim = rot;
    r.table_dtype = code(table_type);
    r.axes = (int32_t)axes;
    if (axes > 1) {
      int64_t i = 0;
      if (interleaved) {  // the axes in turn, as long as each has pairs left
        for (; i < pairs; ++i) pair_axis[i] = i < axes * sections[i % axes] ? (uint8_t)(i % axes) : 0;
      } else {  // runs of pairs
        for (int64_t a = 0; a < axes; ++a)
          for (int64_t n = 0; n < sections[a]; ++n) pair_axis[i++] = (uint8_t)a;
      }
      r.pair_axis = pair_axis.data();
    }
  }
};

Tensor rope_axes_run(const Tensor& x_in, const Tensor& cos, const Tensor& sin, const OptTensor& positions, at::IntArrayRef sections, bool interleaved,
                     int transpose) {
  const int dtype = code(x_in.scalar_type());
  const Rotary rot(x_in, cos, sin, positions, sections, interleaved);
  Tensor out = result_like(x_in);
  if (out.numel() == 0) return out;
  const Tensor x = operand(x_in);
  launch(x, "xg_rope_axes", [&](void* stream) {
    return xg_rope_axes(ptr(x), ptr(out), x.size(0), x.size(1), x.size(2), x.size(3), strides(x), strides(out), &rot.r, transpose, dtype, stream);
  });
  return out;
}
Tensor rope_axes(const Tensor& x, const Tensor& cos, const Tensor& sin, const OptTensor& positions, at::IntArrayRef sections, bool interleaved) {
  return rope_axes_run(x, cos, sin, positions, sections, interleaved, 0);
}
Tensor rope_axes_bwd(const Tensor& gy, const Tensor& cos, const Tensor& sin, const OptTensor& positions, at::IntArrayRef sections, bool interleaved) {
  return rope_axes_run(gy, cos, sin, positions, sections, interleaved, 1);
}

// ------------------------------------------------------- norm and rotation
void check_qk(const Tensor& q, const Tensor& k, const OptTensor& wq, const OptTensor& wk) {
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && q.size(0) == k.size(0) && q.size(2) == k.size(2) && q.size(3) == k.size(3),
                    "qk_norm_rope: q and k must be [B, H, S, D] and [B, Hkv, S, D]");
  TORCH_CHECK_TYPE(q.scalar_type() == k.scalar_type(), "qk_norm_rope: q and k must share a dtype");
  for (const OptTensor* w : {&wq, &wk})
    TORCH_CHECK_VALUE(!has(*w) || ((*w)->dim() == 1 && (*w)->size(0) == q.size(3)), "qk_norm_rope: a weight is one row of the head dim");
  same_device(q, {&wq, &wk});
  TORCH_CHECK_VALUE(q.device() == k.device(), "xpu_ops: tensors on different devices");
}

// The weights as the kernels read them: both in the tensors' dtype or both in fp32.
struct Weights {
  OptTensor q, k;
  at::ScalarType type;
  int dtype;
  Weights(const Tensor& x, const OptTensor& wq, const OptTensor& wk) : type(x.scalar_type()) {
    for (const OptTensor* w : {&wq, &wk})
      if (has(*w) && (*w)->scalar_type() != x.scalar_type()) type = at::kFloat;
    auto prepare = [&](const OptTensor& w) -> OptTensor {
      if (!has(w)) return std::nullopt;
      Tensor t = w->scalar_type() == type ? *w : w->to(type);
      t = t.contiguous();
      return misaligned(t) ? t.clone() : t;
    };
    q = prepare(wq);
    k = prepare(wk);
    dtype = code(type);
  }
};

std::tuple<Tensor, Tensor> qk_norm_rope(const Tensor& q_in, const Tensor& k_in, const OptTensor& wq, const OptTensor& wk, const Tensor& cos,
                                        const Tensor& sin, const OptTensor& positions, at::IntArrayRef sections, bool interleaved, double eps) {
  check_qk(q_in, k_in, wq, wk);
  const int dtype = code(q_in.scalar_type());
  const Rotary rot(q_in, cos, sin, positions, sections, interleaved);
  Tensor q_out = result_like(q_in), k_out = result_like(k_in);
  if (q_out.numel() + k_out.numel() == 0) return {q_out, k_out};
  const Tensor q = operand(q_in), k = operand(k_in);
  const Weights w(q, wq, wk);
  launch(q, "xg_qk_norm_rope", [&](void* stream) {
    return xg_qk_norm_rope(ptr(q), ptr(k), ptr(w.q), ptr(w.k), ptr(q_out), ptr(k_out), q.size(0), q.size(1), k.size(1), q.size(2), q.size(3),
                           strides(q), strides(k), strides(q_out), strides(k_out), &rot.r, (float)eps, dtype, w.dtype, stream);
  });
  return {q_out, k_out};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> qk_norm_rope_bwd(const Tensor& q_in, const Tensor& k_in, const OptTensor& wq, const OptTensor& wk,
                                                            const Tensor& gq_in, const Tensor& gk_in, const Tensor& cos, const Tensor& sin,
                                                            const OptTensor& positions, at::IntArrayRef sections, bool interleaved, double eps,
                                                            bool want_gw) {
  check_qk(q_in, k_in, wq, wk);
  TORCH_CHECK_VALUE(gq_in.sizes() == q_in.sizes() && gk_in.sizes() == k_in.sizes() && gq_in.scalar_type() == q_in.scalar_type() &&
                        gk_in.scalar_type() == q_in.scalar_type() && gq_in.device() == q_in.device() && gk_in.device() == q_in.device(),
                    "qk_norm_rope_bwd: gq and gk must match q and k in shape, dtype and device");
  const int dtype = code(q_in.scalar_type());
  const Rotary rot(q_in, cos, sin, positions, sections, interleaved);
  Tensor dq = result_like(q_in), dk = result_like(k_in);
  auto weight_grad = [&](const OptTensor& w) { return at::empty({want_gw && has(w) ? q_in.size(3) : 0}, has(w) ? w->options() : q_in.options()); };
  Tensor gwq = weight_grad(wq), gwk = weight_grad(wk);
  if (dq.numel() + dk.numel() == 0) return {dq, dk, gwq.zero_(), gwk.zero_()};
  const Tensor q = operand(q_in), k = operand(k_in), gq = operand(gq_in), gk = operand(gk_in);
  const Weights w(q, wq, wk);
  const int64_t B = q.size(0), H = q.size(1), Hkv = k.size(1), S = q.size(2), D = q.size(3);
  // a gradient in a weight's own dtype (any that converts), where the kernel works in fp32 because of it or of the other weight
  auto kernel_grad = [&](const Tensor& g) { return g.numel() && g.scalar_type() != w.type ? at::empty(g.sizes(), g.options().dtype(w.type)) : g; };
  const Tensor kq = kernel_grad(gwq), kk = kernel_grad(gwk);
  const bool any = gwq.numel() || gwk.numel();
  const int64_t n = any ? xg_qk_norm_rope_bwd_workspace_floats(B, H, Hkv, S, D) : 0;
  const Tensor ws = n ? at::empty({n}, q.options().dtype(at::kFloat)) : Tensor();
  launch(q, "xg_qk_norm_rope_bwd", [&](void* stream) {
    return xg_qk_norm_rope_bwd(ptr(q), ptr(k), ptr(w.q), ptr(w.k), ptr(gq), ptr(gk), ptr(dq), ptr(dk), gwq.numel() ? ptr(kq) : nullptr,
                               gwk.numel() ? ptr(kk) : nullptr, n ? ws.data_ptr<float>() : nullptr, n, B, H, Hkv, S, D, strides(q), strides(k),
                               strides(gq), strides(gk), strides(dq), strides(dk), &rot.r, (float)eps, dtype, w.dtype, stream);
  });
  if (!kq.is_same(gwq)) gwq.copy_(kq);
  if (!kk.is_same(gwk)) gwk.copy_(kk);
  return {dq, dk, gwq, gwk};
}

// ---------------------------------------------------------- linear attention
void check_linear(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const OptTensor& state, const OptTensor& lengths) {
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && k.sizes() == v.sizes(), "linear_attn: q must be [B, H, S, D], k and v [B, Hkv, S, D]");
  const int64_t B = q.size(0), H = q.size(1), D = q.size(3), Hkv = k.size(1);
  TORCH_CHECK_VALUE(k.size(0) == B && k.size(2) == q.size(2) && k.size(3) == D && (Hkv ? H % Hkv == 0 : H == 0), "linear_attn: inconsistent q/k/v shapes");
  TORCH_CHECK_VALUE(D == 64 || D == 128, "linear_attn: head dim must be 64 or 128");
  const auto type = q.scalar_type();
  TORCH_CHECK_TYPE((type == at::kBFloat16 || type == at::kHalf) && k.scalar_type() == type && v.scalar_type() == type,
                   "linear_attn: q, k, v must share a dtype, bfloat16 or float16");
  TORCH_CHECK_VALUE(log_decay.dim() == 1 && log_decay.size(0) == H && log_decay.scalar_type() == at::kFloat, "linear_attn: log_decay must be float32 [H]");
  TORCH_CHECK_VALUE(!has(state) || (state->dim() == 4 && state->size(0) == B && state->size(1) == H && state->size(2) == D && state->size(3) == D &&
                                    state->scalar_type() == at::kFloat),
                    "linear_attn: states must be float32 [B, H, D, D]");
  TORCH_CHECK_VALUE(!has(lengths) || (lengths->dim() == 1 && lengths->size(0) == B &&
                                      (lengths->scalar_type() == at::kInt || lengths->scalar_type() == at::kLong)),
                    "linear_attn: lengths must be int32 or int64 [B]");
  same_device(q, {&state, &lengths});
  TORCH_CHECK_VALUE(k.device() == q.device() && v.device() == q.device() && log_decay.device() == q.device(), "xpu_ops: tensors on different devices");
}

OptTensor state_operand(const OptTensor& s) {
  if (!has(s)) return std::nullopt;
  Tensor t = s->contiguous();
  return misaligned(t) ? t.clone(at::MemoryFormat::Contiguous) : t;
}
OptTensor contiguous(const OptTensor& t) { return has(t) ? OptTensor(t->contiguous()) : std::nullopt; }
int wide(const OptTensor& lengths) { return has(lengths) && lengths->scalar_type() == at::kLong; }
Tensor workspace(int64_t floats, const Tensor& like) { return floats ? at::empty({floats}, like.options().dtype(at::kFloat)) : Tensor(); }
float* floats_of(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
float* floats_of(const OptTensor& t) { return has(t) ? t->data_ptr<float>() : nullptr; }

std::tuple<Tensor, Tensor> linear_attn(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& log_decay_in, const OptTensor& state_in,
                                       const OptTensor& lengths_in, double scale) {
  check_linear(q_in, k_in, v_in, log_decay_in, state_in, lengths_in);
  const int64_t B = q_in.size(0), H = q_in.size(1), S = q_in.size(2), D = q_in.size(3), Hkv = k_in.size(1);
  Tensor out = result_like(q_in, kMaxPitch), state_out = at::empty({B, H, D, D}, q_in.options().dtype(at::kFloat));
  if (out.numel() == 0) return {out, has(state_in) ? state_out.copy_(*state_in) : state_out.zero_()};
  const Tensor q = token_operand(q_in), k = token_operand(k_in), v = token_operand(v_in), g = log_decay_in.contiguous();
  const OptTensor state = state_operand(state_in), lengths = contiguous(lengths_in);
  const int64_t n = xg_linear_attn_workspace_floats(B, H, S, D);
  const Tensor ws = workspace(n, q);
  launch(q, "xg_linear_attn", [&](void* stream) {
    return xg_linear_attn(ptr(q), ptr(k), ptr(v), g.data_ptr<float>(), floats_of(state), ptr(lengths), wide(lengths), ptr(out),
                          state_out.data_ptr<float>(), floats_of(ws), n, B, H, Hkv, S, D, strides(q), strides(k), strides(v), strides(out), (float)scale,
                          code(q.scalar_type()), stream);
  });
  return {out, state_out};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> linear_attn_bwd(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& log_decay_in,
                                                           const OptTensor& state_in, const OptTensor& lengths_in, const Tensor& d_out_in,
                                                           const OptTensor& d_state_out_in, double scale, bool want_d_state) {
  check_linear(q_in, k_in, v_in, log_decay_in, state_in, lengths_in);
  const int64_t B = q_in.size(0), H = q_in.size(1), S = q_in.size(2), D = q_in.size(3), Hkv = k_in.size(1);
  TORCH_CHECK_VALUE(d_out_in.sizes() == q_in.sizes() && d_out_in.scalar_type() == q_in.scalar_type() && d_out_in.device() == q_in.device(),
                    "linear_attn_bwd: d_out must match q in shape, dtype and device");
  TORCH_CHECK_VALUE(!has(d_state_out_in) || (d_state_out_in->sizes() == at::IntArrayRef({B, H, D, D}) && d_state_out_in->scalar_type() == at::kFloat &&
                                             d_state_out_in->device() == q_in.device()),
                    "linear_attn_bwd: d_state_out must be float32 [B, H, D, D]");
  Tensor dq = result_like(q_in, kMaxPitch), dk = result_like(k_in, kMaxPitch), dv = result_like(v_in, kMaxPitch);
  const auto fp32 = q_in.options().dtype(at::kFloat);
  Tensor d_state = want_d_state ? at::empty({B, H, D, D}, fp32) : at::empty({0}, fp32);
  if (dq.numel() == 0) {
    if (want_d_state) has(d_state_out_in) ? d_state.copy_(*d_state_out_in) : d_state.zero_();
    return {dq, dk.zero_(), dv.zero_(), d_state};  // (key heads without query heads: sums of nothing)
  }
  const Tensor q = token_operand(q_in), k = token_operand(k_in), v = token_operand(v_in), d_out = token_operand(d_out_in), g = log_decay_in.contiguous();
  const OptTensor state = state_operand(state_in), d_state_out = state_operand(d_state_out_in), lengths = contiguous(lengths_in);
  const int64_t n = xg_linear_attn_bwd_workspace_floats(B, H, Hkv, S, D);
  const Tensor ws = workspace(n, q);
  launch(q, "xg_linear_attn_bwd", [&](void* stream) {
    return xg_linear_attn_bwd(ptr(q), ptr(k), ptr(v), g.data_ptr<float>(), floats_of(state), ptr(lengths), wide(lengths), ptr(d_out),
                              floats_of(d_state_out), ptr(dq), ptr(dk), ptr(dv), want_d_state ? d_state.data_ptr<float>() : nullptr, floats_of(ws), n, B,
                              H, Hkv, S, D, strides(q), strides(k), strides(v), strides(d_out), strides(dq), strides(dk), strides(dv), (float)scale,
                              code(q.scalar_type()), stream);
  });
  return {dq, dk, dv, d_state};
}

Tensor linear_attn_step(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& log_decay_in, Tensor& state, double scale) {
  check_linear(q_in, k_in, v_in, log_decay_in, state, std::nullopt);
  const int64_t B = q_in.size(0), H = q_in.size(1), D = q_in.size(3);
  TORCH_CHECK_VALUE(q_in.size(2) == 1, "linear_attn_step: one token, q [B, H, 1, D]");
  TORCH_CHECK_VALUE(state.stride(3) == 1 && state.stride(2) == D,
                    "linear_attn_step: the [D, D] matrices of the state must be contiguous (it is updated in place)");
  Tensor out = at::empty({B, H, 1, D}, q_in.options());
  if (out.numel() == 0) return out;
  auto unit = [](const Tensor& t) { return t.stride(3) == 1 ? t : t.contiguous(); };
  const Tensor q = unit(q_in), k = unit(k_in), v = unit(v_in), g = log_decay_in.contiguous();
  launch(q, "xg_linear_attn_step", [&](void* stream) {
    return xg_linear_attn_step(ptr(q), ptr(k), ptr(v), g.data_ptr<float>(), state.data_ptr<float>(), ptr(out), B, H, k.size(1), D, strides(q), strides(k),
                               strides(v), strides(out), strides(state), (float)scale, code(q.scalar_type()), stream);
  });
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();  // a graph that saved the state must see that it changed
  return out;
}

// ------------------------------------------------------------------ autograd
// The formulas: each forward and backward goes through the dispatcher, so that a tracer sees the op and its *_bwd op.
template <typename F>
c10::TypedOperatorHandle<F> handle(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

bool wants_grad(std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), "xpu_ops: no forward-mode gradients");
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
Tensor or_undefined(const OptTensor& t) { return has(t) ? *t : Tensor(); }
OptTensor or_none(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

using RopeSig = Tensor(const Tensor&, const Tensor&, const Tensor&, const OptTensor&, at::IntArrayRef, bool);

struct RopeAxes : torch::autograd::Function<RopeAxes> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& cos, const Tensor& sin, const OptTensor& positions, at::IntArrayRef sections,
                        bool interleaved) {
    static const auto op = handle<RopeSig>("xpu_ops::rope_axes");
    ctx->save_for_backward({cos, sin, or_undefined(positions)});
    ctx->saved_data["sections"] = sections.vec();
    ctx->saved_data["interleaved"] = interleaved;
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(x, cos, sin, positions, sections, interleaved);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    static const auto op = handle<RopeSig>("xpu_ops::rope_axes_bwd");
    const auto saved = ctx->get_saved_variables();
    const auto sections = ctx->saved_data["sections"].toIntVector();
    return {op.call(g[0], saved[0], saved[1], or_none(saved[2]), sections, ctx->saved_data["interleaved"].toBool()), Tensor(), Tensor(), Tensor(), Tensor(),
            Tensor()};
  }
};

Tensor rope_axes_autograd(const Tensor& x, const Tensor& cos, const Tensor& sin, const OptTensor& positions, at::IntArrayRef sections, bool interleaved) {
  TORCH_CHECK_NOT_IMPLEMENTED(!wants_grad({&cos, &sin}), "xpu_ops::rope_axes: no gradient for the cos / sin tables");
  if (wants_grad({&x})) return RopeAxes::apply(x, cos, sin, positions, sections, interleaved);
  static const auto op = handle<RopeSig>("xpu_ops::rope_axes");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, cos, sin, positions, sections, interleaved);
}

using QkSig = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, const Tensor&, const Tensor&, const OptTensor&,
                                         at::IntArrayRef, bool, double);
using QkBwdSig = std::tuple<Tensor, Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, const Tensor&, const Tensor&,
                                                            const Tensor&, const Tensor&, const OptTensor&, at::IntArrayRef, bool, double, bool);

struct QkNormRope : torch::autograd::Function<QkNormRope> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const OptTensor& wq, const OptTensor& wk, const Tensor& cos,
                               const Tensor& sin, const OptTensor& positions, at::IntArrayRef sections, bool interleaved, double eps) {
    static const auto op = handle<QkSig>("xpu_ops::qk_norm_rope");
    ctx->save_for_backward({q, k, or_undefined(wq), or_undefined(wk), cos, sin, or_undefined(positions)});
    ctx->saved_data["sections"] = sections.vec();
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["eps"] = eps;
    at::AutoDispatchBelowADInplaceOrView below;
    auto [oq, ok] = op.call(q, k, wq, wk, cos, sin, positions, sections, interleaved, eps);
    return {oq, ok};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    static const auto op = handle<QkBwdSig>("xpu_ops::qk_norm_rope_bwd");
    const auto s = ctx->get_saved_variables();
    const auto sections = ctx->saved_data["sections"].toIntVector();
    // the inputs are numbered without those that are not there
    const bool need_wq = s[2].defined() && ctx->needs_input_grad(2), need_wk = s[3].defined() && ctx->needs_input_grad(s[2].defined() ? 3 : 2);
    auto [dq, dk, gwq, gwk] = op.call(s[0], s[1], or_none(s[2]), or_none(s[3]), g[0], g[1], s[4], s[5], or_none(s[6]), sections,
                                      ctx->saved_data["interleaved"].toBool(), ctx->saved_data["eps"].toDouble(), need_wq || need_wk);
    return {dq, dk, need_wq ? gwq : Tensor(), need_wk ? gwk : Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor> qk_norm_rope_autograd(const Tensor& q, const Tensor& k, const OptTensor& wq, const OptTensor& wk, const Tensor& cos,
                                                 const Tensor& sin, const OptTensor& positions, at::IntArrayRef sections, bool interleaved, double eps) {
  TORCH_CHECK_NOT_IMPLEMENTED(!wants_grad({&cos, &sin}), "xpu_ops::qk_norm_rope: no gradient for the cos / sin tables");
  const Tensor uq = or_undefined(wq), uk = or_undefined(wk);
  if (wants_grad({&q, &k, &uq, &uk})) {
    auto out = QkNormRope::apply(q, k, wq, wk, cos, sin, positions, sections, interleaved, eps);
    return {out[0], out[1]};
  }
  static const auto op = handle<QkSig>("xpu_ops::qk_norm_rope");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(q, k, wq, wk, cos, sin, positions, sections, interleaved, eps);
}

using LinSig = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, double);
using LinBwdSig = std::tuple<Tensor, Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const OptTensor&, const OptTensor&,
                                                             const Tensor&, const OptTensor&, double, bool);
using StepSig = Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&, Tensor&, double);

struct LinearAttn : torch::autograd::Function<LinearAttn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const OptTensor& state,
                               const OptTensor& lengths, double scale) {
    static const auto op = handle<LinSig>("xpu_ops::linear_attn");
    ctx->save_for_backward({q, k, v, log_decay, or_undefined(state), or_undefined(lengths)});
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);  // an unused output hands over nothing: no gradient of the final state is read then
    at::AutoDispatchBelowADInplaceOrView below;
    auto [out, state_out] = op.call(q, k, v, log_decay, state, lengths, scale);
    return {out, state_out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    static const auto op = handle<LinBwdSig>("xpu_ops::linear_attn_bwd");
    variable_list none(7);
    if (!g[0].defined() && !g[1].defined()) return none;
    const auto s = ctx->get_saved_variables();
    const bool want = s[4].defined() && ctx->needs_input_grad(4);
    auto [dq, dk, dv, d_state] = op.call(s[0], s[1], s[2], s[3], or_none(s[4]), or_none(s[5]), g[0].defined() ? g[0] : at::zeros_like(s[0]), or_none(g[1]),
                                         ctx->saved_data["scale"].toDouble(), want);
    return {dq, dk, dv, Tensor(), want ? d_state : Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor> linear_attn_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const OptTensor& state,
                                                const OptTensor& lengths, double scale) {
  TORCH_CHECK_NOT_IMPLEMENTED(!wants_grad({&log_decay}),
                              "xpu_ops::linear_attn: no gradient for log_decay (only q, k, v and the state are differentiable)");
  const Tensor s = or_undefined(state);
  if (wants_grad({&q, &k, &v, &s})) {
    auto out = LinearAttn::apply(q, k, v, log_decay, state, lengths, scale);
    return {out[0], out[1]};
  }
  static const auto op = handle<LinSig>("xpu_ops::linear_attn");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(q, k, v, log_decay, state, lengths, scale);
}

Tensor linear_attn_step_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, Tensor& state, double scale) {
  TORCH_CHECK_NOT_IMPLEMENTED(!wants_grad({&q, &k, &v, &log_decay, &state}),
                              "xpu_ops::linear_attn_step: no gradient (the state is updated in place; use linear_attn to train)");
  static const auto op = handle<StepSig>("xpu_ops::linear_attn_step");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(q, k, v, log_decay, state, scale);
}

}  // namespace

// ROCm devices are "cuda" to PyTorch.
TORCH_LIBRARY_IMPL(xpu_ops, CUDA, m) {
  m.impl("rope_axes", rope_axes);
  m.impl("rope_axes_bwd", rope_axes_bwd);
  m.impl("qk_norm_rope", qk_norm_rope);
  m.impl("qk_norm_rope_bwd", qk_norm_rope_bwd);
  m.impl("linear_attn", linear_attn);
  m.impl("linear_attn_bwd", linear_attn_bwd);
  m.impl("linear_attn_step", linear_attn_step);
}
TORCH_LIBRARY_IMPL(xpu_ops, Autograd, m) {
  m.impl("rope_axes", rope_axes_autograd);
  m.impl("qk_norm_rope", qk_norm_rope_autograd);
  m.impl("linear_attn", linear_attn_autograd);
  m.impl("linear_attn_step", linear_attn_step_autograd);
  // differentiating a gradient again is refused
  m.impl("rope_axes_bwd", torch::autograd::autogradNotImplementedFallback());
  m.impl("qk_norm_rope_bwd", torch::autograd::autogradNotImplementedFallback());
  m.impl("linear_attn_bwd", torch::autograd::autogradNotImplementedFallback());
}
