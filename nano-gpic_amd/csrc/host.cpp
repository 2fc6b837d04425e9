// The host side of the path's calls in one native module (_gpic_host): output allocation and the C-ABI calls of a cast
// group, a GEMM, a weight gradient, the whole forward or backward of a phase-3 linear, and the row-scaled operators, their
// linears as nodes of the autograd graph, without a Python frame, a ctypes conversion and a tensor constructor for each piece.
// A linear of a few hundred rows is bound by that host time, not by its kernels (~40 us of Python for 25 us of kernels in a
// sampler's proj; the row-scaled norm and linear of 331 rows, forward and backward, 165 us with Python Functions and 74-114
// with nodes, for 53 us of kernels).
//
// Every function takes tensors of the usual form only (on the current device, contiguous, 16-byte aligned, the types
// the C ABI takes) and returns None for any other, for which the caller runs its general form. Outputs are ordinary
// tensors of torch's allocator on the current stream, as the general form's. dev, ws, stream: the current device, its
// current stream's cast workspace (0 for the calls that cast nothing) and that stream. The GIL is released while a call
// allocates and launches, as ctypes and torch's own operations release it: a launch waits where the queue is full.
#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <ATen/hip/impl/HIPCachingAllocatorMasqueradingAsCUDA.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <optional>
#include <string>

#include "../../include/gpic_fp8.h"

namespace py = pybind11;

namespace {

constexpr auto kE4 = at::kFloat8_e4m3fn;

void check(int status, const char *what) {
  if (status != GPIC_OK)
    throw std::runtime_error(std::string(what) + " failed: " + gpic_fp8_status_string(status) + " (status " +
                             std::to_string(status) + ")");
}

// Whether t has memory of its own: a fake tensor, or a subclass that wraps others, has none to read.
bool has_memory(const at::Tensor &t) { return !t.key_set().has(c10::DispatchKey::Python); }
bool plain(const at::Tensor &t, int dev) {
  return t.is_cuda() && t.get_device() == dev && has_memory(t) && t.layout() == at::kStrided && t.is_contiguous() &&
         (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0;
}
bool castable(const at::Tensor &t, int dev) {
  return (t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat) && plain(t, dev);
}
// A contiguous [rows, cols] e4m3 operand with 16-byte rows, and its scale
bool operand(const at::Tensor &t, const at::Tensor &s, int dev) {
  return t.scalar_type() == kE4 && t.dim() == 2 && t.size(1) % 16 == 0 && plain(t, dev) && s.scalar_type() == at::kFloat &&
         s.dim() == 1 && s.size(0) == 1 && s.is_cuda() && s.get_device() == dev;
}
int dtype_code(const at::Tensor &t) { return t.scalar_type() == at::kFloat ? GPIC_DTYPE_F32 : GPIC_DTYPE_BF16; }
template <class T>
T *ptr(const at::Tensor &t) {
  return static_cast<T *>(t.data_ptr());
}
// at::empty on like's device, which the callers have checked to be the current one, without the dispatcher's walk to it (a tensor
// 0.5 us instead of 1.0; one token's norm, five tensors, 7.3 us a call instead of 9.3).
at::Tensor make(const at::Tensor & /* like */, at::IntArrayRef size, at::ScalarType ty) {
  return at::Tensor(at::detail::empty_generic(size, c10::hip::HIPCachingAllocatorMasqueradingAsCUDA::get(),
                                              c10::DispatchKeySet(c10::DispatchKey::CUDA), ty, std::nullopt));
}

struct Scratch {   // a GEMM's split-K workspace, when its plan has one
  at::Tensor t;
  size_t bytes;
  Scratch(const at::Tensor &like, int64_t M, int64_t N, int64_t K) : bytes(gpic_fp8_gemm_workspace_bytes(M, N, K)) {
    if (bytes) t = make(like, {(int64_t)bytes}, at::kByte);
  }
  void *p() const { return bytes ? t.data_ptr() : nullptr; }
};

enum { kFlat = 0, kBoth = 1, kTransposed = 2 };
constexpr int kMost = 8;

struct Casts {
  at::Tensor q[kMost], qt[kMost], s[kMost];
};
// xs[i]: castable; kind kBoth / kTransposed: 2-D with a multiple of 16 columns
void cast_group(int n, const at::Tensor *const *xs, const int *kinds, void *ws, void *stream, Casts &o) {
  const void *x[kMost];
  int dt[kMost];
  int64_t rows[kMost], cols[kMost], ldt[kMost];
  uint8_t *q[kMost], *qt[kMost];
  float *s[kMost];
  for (int i = 0; i < n; i++) {
    const at::Tensor &t = *xs[i];
    const bool flat = kinds[i] == kFlat;
    rows[i] = flat ? 1 : t.size(0);
    cols[i] = flat ? t.numel() : t.size(1);
    ldt[i] = flat ? 0 : (rows[i] + 15) / 16 * 16;
    o.q[i] = kinds[i] == kTransposed ? make(t, {0}, kE4) : make(t, t.sizes(), kE4);
    o.qt[i] = flat ? make(t, {0}, kE4) : make(t, {cols[i], ldt[i]}, kE4);
    o.s[i] = make(t, {1}, at::kFloat);
    x[i] = t.data_ptr();
    dt[i] = dtype_code(t);
    q[i] = kinds[i] == kTransposed ? nullptr : ptr<uint8_t>(o.q[i]);
    qt[i] = flat ? nullptr : ptr<uint8_t>(o.qt[i]);
    s[i] = ptr<float>(o.s[i]);
  }
  check(gpic_fp8_cast_group(n, x, dt, rows, cols, q, qt, ldt, s, ws, stream), "gpic_fp8_cast_group");
}

bool bias_ok(const std::optional<at::Tensor> &b, int64_t N, int dev) {
  return !b || (castable(*b, dev) && b->dim() == 1 && b->size(0) == N);
}
// a [M, K], b [N, K] -> bf16(sa sb a b^T) (+ bias) [M, N]
at::Tensor gemm_tn(const at::Tensor &a, const at::Tensor &sa, const at::Tensor &b, const at::Tensor &sb,
                   const std::optional<at::Tensor> &bias, void *stream) {
  const int64_t M = a.size(0), K = a.size(1), N = b.size(0);
  at::Tensor c = make(a, {M, N}, at::kBFloat16);
  const Scratch w(a, M, N, K);
  if (bias && bias->scalar_type() == at::kFloat) {
    check(gpic_fp8_gemm_bias32(ptr<uint8_t>(a), K, ptr<float>(sa), ptr<uint8_t>(b), K, ptr<float>(sb), ptr<float>(*bias),
                               ptr<uint16_t>(c), N, M, N, K, w.p(), w.bytes, stream),
          "gpic_fp8_gemm_bias32");
    return c;
  }
  check(gpic_fp8_gemm(ptr<uint8_t>(a), K, ptr<float>(sa), ptr<uint8_t>(b), K, ptr<float>(sb),
                      bias ? ptr<uint16_t>(*bias) : nullptr, ptr<uint16_t>(c), N, M, N, K, 1, w.p(), w.bytes, stream),
        "gpic_fp8_gemm");
  return c;
}
bool wgrad_ok(const at::Tensor &a, const at::Tensor &b) {
  return a.size(0) == b.size(0) && a.size(0) * std::max(a.size(1), b.size(1)) < (int64_t(1) << 31) &&
         b.size(1) < (1 << 21);
}
// a [K, M], b [K, N] -> bf16(sa sb a^T b) [M, N], as fp32 when f32
at::Tensor gemm_mn(const at::Tensor &a, const at::Tensor &sa, const at::Tensor &b, const at::Tensor &sb, bool f32,
                   void *stream) {
  const int64_t K = a.size(0), M = a.size(1), N = b.size(1);
  at::Tensor c = make(a, {M, N}, f32 ? at::kFloat : at::kBFloat16);
  const Scratch w(a, M, N, K);
  if (f32)
    check(gpic_fp8_gemm_mn_f32(ptr<uint8_t>(a), M, ptr<float>(sa), ptr<uint8_t>(b), N, ptr<float>(sb), ptr<float>(c), N,
                               M, N, K, w.p(), w.bytes, stream),
          "gpic_fp8_gemm_mn_f32");
  else
    check(gpic_fp8_gemm_mn(ptr<uint8_t>(a), M, ptr<float>(sa), ptr<uint8_t>(b), N, ptr<float>(sb), nullptr,
                           ptr<uint16_t>(c), N, M, N, K, w.p(), w.bytes, stream),
          "gpic_fp8_gemm_mn");
  return c;
}

at::Tensor bias_grad(const at::Tensor &dy, bool f32, void *stream) {
  const int64_t M = dy.size(0), N = dy.size(1);
  const size_t bytes = gpic_fp8_bias_grad_workspace_bytes(M, N);
  at::Tensor part = make(dy, {std::max<int64_t>((int64_t)bytes, 16)}, at::kByte);
  at::Tensor db = make(dy, {N}, f32 ? at::kFloat : at::kBFloat16);
  check(gpic_fp8_bias_grad(ptr<uint16_t>(dy), N, M, N, db.data_ptr(), f32 ? GPIC_DTYPE_F32 : GPIC_DTYPE_BF16,
                           part.data_ptr(), bytes, stream),
        "gpic_fp8_bias_grad");
  return db;
}

typedef uintptr_t handle;
void *vp(handle h) { return reinterpret_cast<void *>(h); }
typedef py::gil_scoped_release NoGil;

py::object casts(const std::vector<at::Tensor> &xs, const std::vector<int> &kinds, int dev, handle ws, handle stream) {
  const int n = (int)xs.size();
  if (n < 1 || n > kMost) return py::none();
  const at::Tensor *p[kMost];
  for (int i = 0; i < n; i++) {
    if (!castable(xs[i], dev) || (kinds[i] != kFlat && (xs[i].dim() != 2 || xs[i].size(1) % 16))) return py::none();
    p[i] = &xs[i];
  }
  Casts o;
  {
    NoGil no_gil;
    cast_group(n, p, kinds.data(), vp(ws), vp(stream), o);
  }
  py::list out;
  for (int i = 0; i < n; i++) {
    out.append(o.q[i]);
    out.append(o.qt[i]);
    out.append(o.s[i]);
  }
  return out;
}

py::object gemm(const at::Tensor &a, const at::Tensor &sa, const at::Tensor &b, const at::Tensor &sb,
                const std::optional<at::Tensor> &bias, int dev, handle, handle stream) {
  if (!operand(a, sa, dev) || !operand(b, sb, dev) || a.size(1) != b.size(1) || b.size(0) % 16 ||
      !bias_ok(bias, b.size(0), dev))
    return py::none();
  at::Tensor c;
  {
    NoGil no_gil;
    c = gemm_tn(a, sa, b, sb, bias, vp(stream));
  }
  return py::cast(c);
}

py::object wgrad(const at::Tensor &a, const at::Tensor &sa, const at::Tensor &b, const at::Tensor &sb, bool f32, int dev,
                 handle, handle stream) {
  if (!operand(a, sa, dev) || !operand(b, sb, dev) || !wgrad_ok(a, b)) return py::none();
  at::Tensor c;
  {
    NoGil no_gil;
    c = gemm_mn(a, sa, b, sb, f32, vp(stream));
  }
  return py::cast(c);
}

// x [M, K] bf16, w [N, K], bias [N] or None -> y [M, N], and x's and w's casts: (y, xq, sx, wqt, sw), w's
// transposed bytes only when `both` (else an empty tensor)
py::object linear_fwd(const at::Tensor &x, const at::Tensor &w, const std::optional<at::Tensor> &bias, bool both, int dev,
                      handle ws, handle stream) {
  if (x.dim() != 2 || w.dim() != 2 || x.size(1) != w.size(1) || x.size(1) % 16 || w.size(0) % 16 ||
      !castable(x, dev) || !castable(w, dev) || !bias_ok(bias, w.size(0), dev))
    return py::none();
  const at::Tensor *p[2] = {&x, &w};
  const int kinds[2] = {kFlat, both ? kBoth : kFlat};
  Casts o;
  at::Tensor y;
  {
    NoGil no_gil;
    cast_group(2, p, kinds, vp(ws), vp(stream), o);
    y = gemm_tn(o.q[0], o.s[0], o.q[1], o.s[1], bias, vp(stream));
  }
  return py::make_tuple(y, o.q[0], o.s[0], o.qt[1], o.s[1]);
}

// dy [M, N] bf16, the forward's xq [M, K] and wqt [K, N] -> (dx [M, K], dw [N, K], db [N] or None); dw and db fp32
// (holding bf16 values) when f32, else bf16
py::object linear_bwd(const at::Tensor &dy, const at::Tensor &xq, const at::Tensor &sx, const at::Tensor &wqt,
                      const at::Tensor &sw, bool has_bias, bool f32, int dev, handle ws, handle stream) {
  if (dy.dim() != 2 || dy.scalar_type() != at::kBFloat16 || !plain(dy, dev) || dy.size(1) % 16 ||
      !operand(xq, sx, dev) || !operand(wqt, sw, dev) || wqt.size(0) % 16 || wqt.size(1) != dy.size(1) ||
      xq.size(0) != dy.size(0) || !wgrad_ok(dy, xq))
    return py::none();
  const at::Tensor *p[1] = {&dy};
  const int kinds[1] = {kFlat};
  at::Tensor dx, dw, db;
  {
    NoGil no_gil;
    Casts o;
    cast_group(1, p, kinds, vp(ws), vp(stream), o);
    const at::Tensor &dyq = o.q[0], &sdy = o.s[0];
    dx = gemm_tn(dyq, sdy, wqt, sw, std::nullopt, vp(stream));
    dw = gemm_mn(dyq, sdy, xq, sx, f32, vp(stream));
    if (has_bias) db = bias_grad(dy, f32, vp(stream));
  }
  if (!has_bias) return py::make_tuple(dx, dw, py::none());
  return py::make_tuple(dx, dw, db);
}

// ------------------------------------------------------------------------------------------- row-scaled operators

constexpr int64_t kRowsMaxNorm = 16384, kRowsMaxCast = 32768;   // the C ABI's widest rows
typedef std::optional<at::Tensor> opt;

bool bf16(const at::Tensor &t, int dev) { return t.scalar_type() == at::kBFloat16 && plain(t, dev); }
// A vector of n bf16 or fp32
bool vector_ok(const at::Tensor &t, int64_t n, int dev) { return castable(t, dev) && t.dim() == 1 && t.size(0) == n; }
bool scales_ok(const opt &s, int64_t n, int dev) {
  return !s || (s->scalar_type() == at::kFloat && plain(*s, dev) && s->numel() == n);
}
uint16_t *u16(const opt &t) { return t ? ptr<uint16_t>(*t) : nullptr; }
at::Tensor none_of(const at::Tensor &like, at::ScalarType ty) { return make(like, {0}, ty); }
// Whether a call on these records a gradient, or carries a forward-mode one: the operators themselves have none, and the
// general form says so.
bool records(std::initializer_list<const opt *> ts) {
  const bool on = c10::GradMode::is_enabled();
  for (const opt *t : ts)
    if (*t && ((on && (*t)->requires_grad()) || (*t)->_fw_grad(0).defined())) return true;
  return false;
}

// The temporary tensors of one call as parts of one allocation.
struct Arena {
  size_t n = 0;
  at::Tensor t;
  size_t add(size_t bytes) {
    const size_t at = n;
    n += (bytes + 255) & ~size_t(255);
    return at;
  }
  void make_like(const at::Tensor &like) { t = make(like, {(int64_t)std::max<size_t>(n, 16)}, at::kByte); }
  template <class T>
  T *at(size_t offset) const {
    return reinterpret_cast<T *>(static_cast<uint8_t *>(t.data_ptr()) + offset);
  }
};

// Modulation rows [B, 1, C], [B, C] or [C] bf16: base, row stride and B; false for a form that the general path copies. batch:
// x's first extent where x has a batch (B is then that or 1), else 0 (B divides the rows).
struct Mod {
  const uint16_t *p = nullptr;
  int64_t ld = 0, B = 0;
};
bool mod_ok(const opt &t, int64_t C, int64_t batch, int64_t rows, int dev, Mod &m) {
  if (!t) return true;
  const int64_t d = t->dim();
  if (d < 1 || d > 3 || t->scalar_type() != at::kBFloat16 || !t->is_cuda() || t->get_device() != dev || !has_memory(*t) ||
      t->layout() != at::kStrided || t->size(d - 1) != C || t->stride(d - 1) != 1 || (d == 3 && t->size(1) != 1))
    return false;
  m.B = d == 1 ? 1 : t->size(0);
  m.ld = m.B > 1 ? t->stride(0) : C;
  m.p = ptr<uint16_t>(*t);
  if (m.B < 1 || (m.B != 1 && (batch ? m.B != batch : rows % m.B)) || m.ld % 8 || m.ld < C) return false;
  return (reinterpret_cast<uintptr_t>(m.p) & 15u) == 0;
}

bool row_castable(const at::Tensor &x, int dev) {
  return castable(x, dev) && x.dim() >= 1 && x.size(-1) > 0 && x.size(-1) % 8 == 0 && x.size(-1) <= kRowsMaxCast;
}
bool operand_rows(const at::Tensor &t, int dev) {
  return t.scalar_type() == kE4 && t.dim() == 2 && t.size(1) > 0 && t.size(1) % 16 == 0 && plain(t, dev);
}

struct NormIn {
  Mod gate, shift, scale;
  int64_t ntok = 1;
};
bool norm_ok(const at::Tensor &x, const at::Tensor &w, const opt &a, const opt &gate, const opt &shift, const opt &scale,
             int dev, NormIn &in) {
  if (x.dim() < 2 || !bf16(x, dev)) return false;
  const int64_t C = x.size(-1);
  if (C <= 0 || C % 8 || C > kRowsMaxNorm) return false;
  const int64_t M = x.numel() / C, batch = x.dim() > 2 ? x.size(0) : 0;
  if (M < 1 || !vector_ok(w, C, dev) || (a && (!bf16(*a, dev) || a->sizes() != x.sizes())) || (gate && !a) ||
      shift.has_value() != scale.has_value() || !mod_ok(gate, C, batch, M, dev, in.gate) ||
      !mod_ok(shift, C, batch, M, dev, in.shift) || !mod_ok(scale, C, batch, M, dev, in.scale))
    return false;
  int64_t B = 0;
  for (const Mod *m : {&in.gate, &in.shift, &in.scale})
    if (m->B) {
      if (B && B != m->B) return false;
      B = m->B;
    }
  in.ntok = B ? M / B : 1;
  return true;
}
struct NormOut {
  at::Tensor xn, h, rstd;
};
// q, s: where the bytes and scales go; weight (or none) -> wq, sw in the same launch
NormOut norm_run(const at::Tensor &x, const at::Tensor &w, double eps, const opt &a, const NormIn &in, bool want_h, uint8_t *q,
                 float *s, const at::Tensor *weight, uint8_t *wq, float *sw, void *stream) {
  const int64_t C = x.size(-1), M = x.numel() / C;
  NormOut o;
  o.xn = a ? make(x, x.sizes(), at::kBFloat16) : none_of(x, at::kBFloat16);
  o.h = want_h ? make(x, x.sizes(), at::kBFloat16) : none_of(x, at::kBFloat16);
  o.rstd = make(x, {M}, at::kFloat);
  check(gpic_fp8_rmsnorm_rows(ptr<uint16_t>(x), C, u16(a), C, in.gate.p, in.gate.ld, w.data_ptr(), dtype_code(w), in.shift.p,
                              in.shift.ld, in.scale.p, in.scale.ld, M, in.ntok, C, (float)eps,
                              a ? ptr<uint16_t>(o.xn) : nullptr, want_h ? ptr<uint16_t>(o.h) : nullptr, ptr<float>(o.rstd), q,
                              s, weight ? weight->data_ptr() : nullptr, weight ? dtype_code(*weight) : 0,
                              weight ? weight->size(0) : 0, wq, sw, stream),
        "gpic_fp8_rmsnorm_rows");
  return o;
}

struct GemmIn {
  const uint8_t *a, *b;
  const float *sa, *sb;
  int64_t M, N, K;
  const opt *bias = nullptr;
  int act = GPIC_ACT_NONE;
  const uint16_t *res = nullptr;
  Mod gate;
};
// y [M, N] (SwiGLU: N / 2), z [M, N] or null; ws: gpic_fp8_gemm_workspace_bytes(M, N, K)
void gemm_rows_call(const GemmIn &g, uint16_t *y, uint16_t *z, void *ws, size_t bytes, void *stream) {
  const int64_t No = g.act == GPIC_ACT_SWIGLU ? g.N / 2 : g.N;
  const bool b = g.bias && *g.bias;
  check(gpic_fp8_gemm_rows(g.a, g.K, g.sa, g.b, g.K, g.sb, b ? (*g.bias)->data_ptr() : nullptr, b ? dtype_code(**g.bias) : 0,
                           g.act, g.res, No, g.gate.p, g.gate.ld, g.gate.B ? g.M / g.gate.B : 1, y, No, z, g.N, g.M, g.N, g.K,
                           bytes ? ws : nullptr, bytes, stream),
        "gpic_fp8_gemm_rows");
}

py::object cast_rows(const at::Tensor &x, int dev, handle, handle stream) {
  const opt ox = x;
  if (!row_castable(x, dev) || records({&ox})) return py::none();
  const int64_t C = x.size(-1), M = x.numel() / C;
  at::Tensor q, s;
  {
    NoGil no_gil;
    q = make(x, x.sizes(), kE4);
    s = make(x, {M}, at::kFloat);
    check(gpic_fp8_tcast_rows(x.data_ptr(), dtype_code(x), C, M, C, ptr<uint8_t>(q), ptr<float>(s), nullptr, 0, 0, 0, nullptr,
                              nullptr, vp(stream)),
          "gpic_fp8_tcast_rows");
  }
  return py::make_tuple(q, s);
}

py::object norm_rows(const at::Tensor &x, const at::Tensor &w, double eps, const opt &a, const opt &gate, const opt &shift,
                     const opt &scale, bool want_h, int dev, handle, handle stream) {
  NormIn in;
  const opt ox = x, ow = w;
  if (!norm_ok(x, w, a, gate, shift, scale, dev, in) || records({&ox, &ow, &a, &gate, &shift, &scale})) return py::none();
  NormOut o;
  at::Tensor q, s;
  {
    NoGil no_gil;
    q = make(x, x.sizes(), kE4);
    s = make(x, {x.numel() / x.size(-1)}, at::kFloat);
    o = norm_run(x, w, eps, a, in, want_h, ptr<uint8_t>(q), ptr<float>(s), nullptr, nullptr, nullptr, vp(stream));
  }
  return py::make_tuple(o.xn, o.h, q, s, o.rstd);
}

py::object gemm_rows(const at::Tensor &a, const opt &sa, const at::Tensor &b, const opt &sb, const opt &bias, int act,
                     const opt &res, const opt &gate, bool want_z, int dev, handle, handle stream) {
  const opt oa = a, ob = b;
  if (!operand_rows(a, dev) || !operand_rows(b, dev) || a.size(1) != b.size(1)) return py::none();
  const int64_t M = a.size(0), K = a.size(1), N = b.size(0), No = act == GPIC_ACT_SWIGLU ? N / 2 : N;
  GemmIn g{ptr<uint8_t>(a), ptr<uint8_t>(b), sa ? ptr<float>(*sa) : nullptr, sb ? ptr<float>(*sb) : nullptr, M, N, K,
           &bias, act, u16(res)};
  if (M < 1 || N < 16 || N % (act == GPIC_ACT_SWIGLU ? 32 : 16) || !scales_ok(sa, M, dev) || !scales_ok(sb, N, dev) ||
      !bias_ok(bias, N, dev) || (res && (!bf16(*res, dev) || res->dim() != 2 || res->size(0) != M || res->size(1) != No)) ||
      !mod_ok(gate, No, 0, M, dev, g.gate) || records({&oa, &sa, &ob, &sb, &bias, &res, &gate}))
    return py::none();
  at::Tensor y, z;
  {
    NoGil no_gil;
    y = make(a, {M, No}, at::kBFloat16);
    z = want_z ? make(a, {M, N}, at::kBFloat16) : none_of(a, at::kBFloat16);
    const Scratch w(a, M, N, K);
    gemm_rows_call(g, ptr<uint16_t>(y), want_z ? ptr<uint16_t>(z) : nullptr, w.p(), w.bytes, vp(stream));
  }
  return py::make_tuple(y, z);
}

bool norm_bwd_ok(int64_t M, const opt &dxn, const at::Tensor &xs, const at::Tensor &w, const at::Tensor &rstd, int dev) {
  if (xs.dim() < 1 || !bf16(xs, dev)) return false;
  const int64_t C = xs.size(-1);
  return C > 0 && C % 8 == 0 && C <= kRowsMaxNorm && xs.numel() == M * C && vector_ok(w, C, dev) &&
         (!dxn || (bf16(*dxn, dev) && dxn->sizes() == xs.sizes())) && scales_ok(rstd, M, dev);
}
py::object norm_rows_bwd(const at::Tensor &dh, const opt &dxn, const at::Tensor &xs, const at::Tensor &w,
                         const at::Tensor &rstd, int dev, handle, handle stream) {
  const opt odh = dh, oxs = xs, ow = w, ors = rstd;
  if (xs.dim() < 1 || xs.size(-1) <= 0 || !bf16(dh, dev) || dh.sizes() != xs.sizes() ||
      !norm_bwd_ok(xs.numel() / xs.size(-1), dxn, xs, w, rstd, dev) || records({&odh, &dxn, &oxs, &ow, &ors}))
    return py::none();
  const int64_t C = xs.size(-1), M = xs.numel() / C;
  at::Tensor dx, dw;
  {
    NoGil no_gil;
    dx = make(xs, xs.sizes(), at::kBFloat16);
    dw = make(xs, {C}, w.scalar_type());
    const size_t bytes = gpic_fp8_rmsnorm_rows_bwd_workspace_bytes(M, C);
    const at::Tensor ws = make(xs, {std::max<int64_t>((int64_t)bytes, 16)}, at::kByte);
    check(gpic_fp8_rmsnorm_rows_bwd(ptr<uint16_t>(dh), u16(dxn), ptr<uint16_t>(xs), w.data_ptr(), dtype_code(w),
                                    ptr<float>(rstd), M, C, ptr<uint16_t>(dx), dw.data_ptr(), dtype_code(dw), ws.data_ptr(),
                                    bytes, vp(stream)),
          "gpic_fp8_rmsnorm_rows_bwd");
  }
  return py::make_tuple(dx, dw);
}

bool rows_weight_ok(const at::Tensor &w, int64_t K, int dev) {
  return w.dim() == 2 && w.size(1) == K && w.size(0) >= 16 && w.size(0) % 16 == 0 && K % 16 == 0 && row_castable(w, dev);
}

// A linear's tensors: x [..., K] or the norm's input, w [N, K]; y [..., N], z [M, N] (or empty), w's bytes and scales.
struct LinearOut {
  at::Tensor y, z, wq, sw;
};
LinearOut linear_out(const at::Tensor &x, const at::Tensor &w, bool want_z) {
  std::vector<int64_t> size = x.sizes().vec();
  size.back() = w.size(0);
  LinearOut o;
  o.y = make(x, size, at::kBFloat16);
  o.z = want_z ? make(x, {x.numel() / x.size(-1), w.size(0)}, at::kBFloat16) : none_of(x, at::kBFloat16);
  o.wq = make(w, w.sizes(), kE4);
  o.sw = make(w, {w.size(0)}, at::kFloat);
  return o;
}
LinearOut linear_run(const at::Tensor &x, const at::Tensor &w, const opt &bias, int act, const opt &res, bool want_z,
                     void *stream) {
  const int64_t K = x.size(-1), M = x.numel() / K, N = w.size(0);
  LinearOut o = linear_out(x, w, want_z);
  Arena m;
  const size_t bytes = gpic_fp8_gemm_workspace_bytes(M, N, K), q = m.add(M * K), s = m.add(4 * M), ws = m.add(bytes);
  m.make_like(x);
  check(gpic_fp8_tcast_rows(x.data_ptr(), GPIC_DTYPE_BF16, K, M, K, m.at<uint8_t>(q), m.at<float>(s), w.data_ptr(),
                            dtype_code(w), K, N, ptr<uint8_t>(o.wq), ptr<float>(o.sw), stream),
        "gpic_fp8_tcast_rows");
  const GemmIn g{m.at<uint8_t>(q), ptr<uint8_t>(o.wq), m.at<float>(s), ptr<float>(o.sw), M, N, K, &bias, act, u16(res)};
  gemm_rows_call(g, ptr<uint16_t>(o.y), want_z ? ptr<uint16_t>(o.z) : nullptr, m.at<uint8_t>(ws), bytes, stream);
  return o;
}
// The norm and the linear that reads its bytes.
std::pair<NormOut, LinearOut> norm_linear_run(const at::Tensor &x, const at::Tensor &wn, double eps, const opt &a,
                                              const NormIn &in, const at::Tensor &w, const opt &bias, int act, bool want_h,
                                              bool want_z, void *stream) {
  const int64_t K = x.size(-1), M = x.numel() / K, N = w.size(0);
  LinearOut o = linear_out(x, w, want_z);
  Arena m;
  const size_t bytes = gpic_fp8_gemm_workspace_bytes(M, N, K), q = m.add(M * K), s = m.add(4 * M), ws = m.add(bytes);
  m.make_like(x);
  NormOut n = norm_run(x, wn, eps, a, in, want_h, m.at<uint8_t>(q), m.at<float>(s), &w, ptr<uint8_t>(o.wq), ptr<float>(o.sw),
                       stream);
  const GemmIn g{m.at<uint8_t>(q), ptr<uint8_t>(o.wq), m.at<float>(s), ptr<float>(o.sw), M, N, K, &bias, act};
  gemm_rows_call(g, ptr<uint16_t>(o.y), want_z ? ptr<uint16_t>(o.z) : nullptr, m.at<uint8_t>(ws), bytes, stream);
  return {n, o};
}

// (x_new or empty, h as bf16 or empty, rstd, y, z or empty, w's bytes, scales)
py::object norm_linear_rows_fwd(const at::Tensor &x, const at::Tensor &wn, double eps, const opt &a, const opt &gate,
                                const opt &shift, const opt &scale, const at::Tensor &w, const opt &bias, int act, bool want_h,
                                bool want_z, int dev, handle, handle stream) {
  NormIn in;
  if (!norm_ok(x, wn, a, gate, shift, scale, dev, in) || !rows_weight_ok(w, x.size(-1), dev) || !bias_ok(bias, w.size(0), dev))
    return py::none();
  std::pair<NormOut, LinearOut> r;
  {
    NoGil no_gil;
    r = norm_linear_run(x, wn, eps, a, in, w, bias, act, want_h, want_z, vp(stream));
  }
  const auto &[n, o] = r;
  return py::make_tuple(n.xn, n.h, n.rstd, o.y, o.z, o.wq, o.sw);
}

struct LinearGrads {
  at::Tensor dx, dw, db;
};
struct BwdIn {
  const at::Tensor &dy, &z, &wq, &sw, &x;
  int act;
  bool need_dx, need_dw, need_db, w32, b32;   // (w32, b32: an fp32 weight's, bias's gradient)
};
bool linear_bwd_ok(const BwdIn &in, int dev) {
  if (in.dy.dim() != 2 || !bf16(in.dy, dev) || !operand_rows(in.wq, dev)) return false;
  const int64_t M = in.dy.size(0), N = in.dy.size(1), K = in.wq.size(1);
  return M >= 1 && N >= 16 && N % 16 == 0 && N <= kRowsMaxCast && in.wq.size(0) == N && scales_ok(in.sw, N, dev) &&
         (in.act == GPIC_ACT_NONE || (bf16(in.z, dev) && in.z.sizes() == in.dy.sizes())) &&
         (!in.need_dw || (bf16(in.x, dev) && in.x.numel() == M * K)) && 2 * M * std::max(N, K) < (int64_t(1) << 31) && K < (1 << 21);
}
// The parts of a linear's backward in its call's arena, and the bytes of its workspaces.
struct BwdParts {
  size_t q, s, dz, qt, ws, b_db, b_dx, b_dw;
};
BwdParts linear_bwd_parts(const BwdIn &in, Arena &m) {
  const int64_t M = in.dy.size(0), N = in.dy.size(1), K = in.wq.size(1);
  BwdParts p;
  p.q = m.add(M * N);
  p.s = m.add(4 * M);
  p.dz = in.act == GPIC_ACT_NONE ? 0 : m.add(2 * M * N);
  p.qt = in.need_dx ? m.add(K * N) : 0;
  p.b_db = in.need_db ? gpic_fp8_act_bwd_rows_workspace_bytes(M, N) : 0;
  p.b_dx = in.need_dx ? gpic_fp8_gemm_workspace_bytes(M, K, N) : 0;
  p.b_dw = in.need_dw ? gpic_fp8_gemm_workspace_bytes(N, K, 2 * M) : 0;   // (planned as an e4m3 GEMM of as many K bytes)
  p.ws = m.add(std::max(p.b_db, std::max(p.b_dx, p.b_dw)));               // (one after the other on one stream)
  return p;
}
// dx: where the input's gradient goes (need_dx), or null: to a tensor of its own
LinearGrads linear_bwd_run(const BwdIn &in, const BwdParts &p, const Arena &m, uint16_t *dx, void *stream) {
  const int64_t M = in.dy.size(0), N = in.dy.size(1), K = in.wq.size(1);
  LinearGrads o;
  const bool on = in.act != GPIC_ACT_NONE;
  uint16_t *dz = on ? m.at<uint16_t>(p.dz) : ptr<uint16_t>(in.dy);
  void *ws = m.at<uint8_t>(p.ws);
  if (in.need_db) o.db = make(in.dy, {N}, in.b32 ? at::kFloat : at::kBFloat16);
  check(gpic_fp8_act_bwd_rows(ptr<uint16_t>(in.dy), N, on ? ptr<uint16_t>(in.z) : nullptr, N, in.act, ptr<float>(in.sw), M, N,
                              on ? dz : nullptr, m.at<uint8_t>(p.q), m.at<float>(p.s),
                              in.need_dx ? ptr<uint8_t>(in.wq) : nullptr, K, in.need_dx ? m.at<uint8_t>(p.qt) : nullptr, N,
                              in.need_db ? o.db.data_ptr() : nullptr, in.b32 ? GPIC_DTYPE_F32 : GPIC_DTYPE_BF16,
                              in.need_db ? ws : nullptr, p.b_db, stream),
        "gpic_fp8_act_bwd_rows");
  if (in.need_dx) {
    if (!dx) {
      o.dx = make(in.dy, {M, K}, at::kBFloat16);
      dx = ptr<uint16_t>(o.dx);
    }
    const GemmIn g{m.at<uint8_t>(p.q), m.at<uint8_t>(p.qt), m.at<float>(p.s), nullptr, M, K, N};
    gemm_rows_call(g, dx, nullptr, ws, p.b_dx, stream);
  }
  if (in.need_dw) {
    o.dw = make(in.dy, {N, K}, in.w32 ? at::kFloat : at::kBFloat16);
    check(gpic_fp8_bf16_gemm_mn(dz, N, ptr<uint16_t>(in.x), K, o.dw.data_ptr(), in.w32 ? GPIC_DTYPE_F32 : GPIC_DTYPE_BF16, K, N,
                                K, M, p.b_dw ? ws : nullptr, p.b_dw, stream),
          "gpic_fp8_bf16_gemm_mn");
  }
  return o;
}
py::object or_none(const at::Tensor &t) { return t.defined() ? py::cast(t) : py::none(); }

// dy [M, N] bf16, the forward's z, w's bytes and scales and x [M, K] bf16 -> (dx [M, K], dw [N, K], db [N]), None where not needed
py::object linear_rows_bwd(const at::Tensor &dy, const at::Tensor &z, int act, const at::Tensor &wq, const at::Tensor &sw,
                           const at::Tensor &x, bool need_dx, bool need_dw, bool need_db, bool w32, bool b32, int dev, handle,
                           handle stream) {
  const BwdIn in{dy, z, wq, sw, x, act, need_dx, need_dw, need_db, w32, b32};
  if (!linear_bwd_ok(in, dev)) return py::none();
  LinearGrads o;
  {
    NoGil no_gil;
    Arena m;
    const BwdParts p = linear_bwd_parts(in, m);
    m.make_like(dy);
    o = linear_bwd_run(in, p, m, nullptr, vp(stream));
  }
  return py::make_tuple(or_none(o.dx), or_none(o.dw), or_none(o.db));
}

// ---- the row-scaled linears in their usual form as nodes of the graph: the calls that the Python Functions of
// gpic_fp8/rows.py make, without a Python frame on either of the engine's threads.

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// An output's gradient as the kernels take it: [M, N] bf16, contiguous, 16-byte aligned.
at::Tensor usual(const at::Tensor &g, int64_t N) {
  at::Tensor t = g.reshape({-1, N}).to(at::kBFloat16).contiguous();
  return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) ? t.clone() : t;
}
// The current stream of t's device: in a backward the engine has made the forward's current.
void *current_stream(const at::Tensor &t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
// The gradients as they are; in a backward that is itself recorded, as outputs of a node that refuses to be differentiated, where
// an output's gradient is of the graph, else as constants, with a warning where they are not (torch's once_differentiable too
// returns constants then, without a word: a term made of them is lost from a sum whose other terms have a gradient).
variable_list once(const variable_list &out, variable_list grads, bool constant = false) {
  bool recorded = false;
  if (!c10::GradMode::is_enabled()) return grads;
  for (const auto &g : out) recorded = recorded || (g.defined() && g.requires_grad());
  if (!recorded && !constant)
    TORCH_WARN("the row-scaled linears are differentiable once: the gradients of a backward under create_graph=True do not "
               "require a gradient, and a loss made of them has none through these linears");
  if (!recorded) return grads;
  struct Refuse : torch::autograd::Node {
    using Node::Node;
    variable_list apply(variable_list &&) override {
      throw std::runtime_error("the row-scaled linears are differentiable once");
    }
  };
  const std::shared_ptr<Refuse> node(new Refuse(torch::autograd::collect_next_edges(out)), torch::autograd::deleteNode);
  for (auto &g : grads)
    if (g.defined()) torch::autograd::set_history(g = g.detach(), node);
  return grads;
}
// Saved tensors come back through the user's hooks, where there are any: on another device, or in another layout.
void saved_ok(bool ok) {
  if (!ok) throw std::runtime_error("the row-scaled linears' backward needs the tensors that the forward saved, as they were saved");
}
// What a node keeps beside its tensors, in one number.
enum : int64_t { kActMask = 7, kFlagW32 = 8, kFlagB32 = 16, kFlagBias = 32, kFlagMore = 64 };   // (more: residual, or a)
int64_t node_flags(int64_t act, const at::Tensor &w, const opt &bias, bool more) {
  return act | (w.scalar_type() == at::kFloat ? kFlagW32 : 0) | (bias ? kFlagBias : 0) |
         (bias && bias->scalar_type() == at::kFloat ? kFlagB32 : 0) | (more ? kFlagMore : 0);
}

struct LinearNode : torch::autograd::Function<LinearNode> {
  // (the order of the arguments is the order of backward's gradients; a tensor that is not there has no edge)
  static at::Tensor forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &w, const opt &bias, const opt &res,
                            int64_t act) {
    const LinearOut o = linear_run(x, w, bias, (int)act, res, act != GPIC_ACT_NONE, current_stream(x));
    ctx->save_for_backward({x, o.z, o.wq, o.sw});
    ctx->set_materialize_grads(false);
    ctx->saved_data["flags"] = node_flags(act, w, bias, res.has_value());
    return o.y;
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &out) {
    variable_list g(5);
    if (!out[0].defined()) return g;
    const variable_list s = ctx->get_saved_variables();
    const at::Tensor &x = s[0], &z = s[1], &wq = s[2], &sw = s[3];
    const int64_t f = ctx->saved_data["flags"].toInt();
    size_t edge = 2;
    const bool db = f & kFlagBias && ctx->needs_input_grad(edge++), dres = f & kFlagMore && ctx->needs_input_grad(edge);
    {
      at::AutoGradMode off(false);
      const at::Tensor dy = usual(out[0], wq.size(0));
      const BwdIn in{dy, z, wq, sw, x, (int)(f & kActMask), ctx->needs_input_grad(0), ctx->needs_input_grad(1), db,
                     (f & kFlagW32) != 0, (f & kFlagB32) != 0};
      saved_ok(linear_bwd_ok(in, dy.get_device()));
      if (in.need_dx || in.need_dw || in.need_db) {
        Arena m;
        const BwdParts p = linear_bwd_parts(in, m);
        m.make_like(dy);
        if (in.need_dx) g[0] = make(x, x.sizes(), at::kBFloat16);
        const LinearGrads o = linear_bwd_run(in, p, m, in.need_dx ? ptr<uint16_t>(g[0]) : nullptr, current_stream(dy));
        g[1] = o.dw;
        g[2] = o.db;
      }
    }
    const bool only_res = !(ctx->needs_input_grad(0) || ctx->needs_input_grad(1) || db);
    if (dres) g[3] = out[0];
    return once(out, std::move(g), only_res);
  }
};

struct NormLinearNode : torch::autograd::Function<NormLinearNode> {
  // (x_new, y), or y alone without a
  static variable_list forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &wn, const at::Tensor &w,
                               const opt &a, const opt &bias, double eps, int64_t act) {
    const auto [n, o] = norm_linear_run(x, wn, eps, a, NormIn(), w, bias, (int)act, w.requires_grad(), act != GPIC_ACT_NONE,
                                        current_stream(x));
    ctx->save_for_backward({a ? n.xn : x, wn, n.rstd, n.h, o.z, o.wq, o.sw});
    ctx->set_materialize_grads(false);
    ctx->saved_data["flags"] = node_flags(act, w, bias, a.has_value());
    if (a) return {n.xn, o.y};
    return {o.y};
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &out) {
    variable_list g(7);
    const int64_t f = ctx->saved_data["flags"].toInt();
    const bool has_a = f & kFlagMore;
    const at::Tensor &dxn_ = has_a ? out[0] : at::Tensor(), &dy_ = out[has_a ? 1 : 0];
    if (!dy_.defined() && !dxn_.defined()) return g;
    const variable_list s = ctx->get_saved_variables();
    const at::Tensor &xs = s[0], &wn = s[1], &rstd = s[2], &h = s[3], &z = s[4], &wq = s[5], &sw = s[6];
    size_t edge = 3;
    const bool da = has_a && ctx->needs_input_grad(edge++), db = f & kFlagBias && ctx->needs_input_grad(edge);
    const bool dx = ctx->needs_input_grad(0), dwn = ctx->needs_input_grad(1), dw = ctx->needs_input_grad(2),
               below = dx || da || dwn;
    {
      at::AutoGradMode off(false);
      const int64_t K = wq.size(1), M = xs.numel() / K, N = wq.size(0);
      const opt dxn = dxn_.defined() ? opt(usual(dxn_, K).view(xs.sizes())) : std::nullopt;
      if (!dy_.defined()) {   // (x_new alone was used: its gradient as it is, and zeros that no value of h or z can spoil)
        if (dx) g[0] = *dxn;
        if (da) g[3] = *dxn;
        if (dwn) g[1] = at::zeros({K}, dxn->options().dtype(wn.scalar_type()));
        if (dw) g[2] = at::zeros({N, K}, dxn->options().dtype(f & kFlagW32 ? at::kFloat : at::kBFloat16));
        if (db) g[4] = at::zeros({N}, dxn->options().dtype(f & kFlagB32 ? at::kFloat : at::kBFloat16));
        return once(out, std::move(g), true);
      }
      const at::Tensor dy = usual(dy_, N);
      const BwdIn in{dy, z, wq, sw, h, (int)(f & kActMask), below, dw, db, (f & kFlagW32) != 0, (f & kFlagB32) != 0};
      saved_ok(linear_bwd_ok(in, dy.get_device()) && (!below || norm_bwd_ok(M, dxn, xs, wn, rstd, dy.get_device())));
      Arena m;
      const BwdParts p = linear_bwd_parts(in, m);
      const size_t bytes = below ? gpic_fp8_rmsnorm_rows_bwd_workspace_bytes(M, K) : 0, dh = below ? m.add(2 * M * K) : 0,
                   ws = m.add(bytes);
      m.make_like(dy);
      void *stream = current_stream(dy);
      const LinearGrads o = linear_bwd_run(in, p, m, below ? m.at<uint16_t>(dh) : nullptr, stream);
      g[2] = o.dw;
      g[4] = o.db;
      if (below) {
        const at::Tensor d = make(xs, xs.sizes(), at::kBFloat16), dn = make(xs, {K}, wn.scalar_type());
        check(gpic_fp8_rmsnorm_rows_bwd(m.at<uint16_t>(dh), u16(dxn), ptr<uint16_t>(xs), wn.data_ptr(), dtype_code(wn),
                                        ptr<float>(rstd), M, K, ptr<uint16_t>(d), dn.data_ptr(), dtype_code(dn),
                                        m.at<uint8_t>(ws), bytes, stream),
              "gpic_fp8_rmsnorm_rows_bwd");
        if (dx) g[0] = d;
        if (da) g[3] = d;
        if (dwn) g[1] = dn;
      }
    }
    return once(out, std::move(g));
  }
};

// Whether the backward takes these sizes (linear_bwd_ok's, from the forward's side).
bool trainable(int64_t M, int64_t N, int64_t K) {
  return N <= kRowsMaxCast && 2 * M * std::max(N, K) < (int64_t(1) << 31) && K < (1 << 21);
}

// residual + act(x w^T + bias), x [..., K] bf16, w [N, K], residual [..., N] bf16; a node of the graph where it records
py::object linear_rows(const at::Tensor &x, const at::Tensor &w, const opt &bias, int act, const opt &res, int dev, handle,
                       handle stream) {
  const opt ox = x, ow = w;
  if (x.dim() < 1 || x.numel() < 1 || !bf16(x, dev) || !row_castable(x, dev) || !rows_weight_ok(w, x.size(-1), dev) ||
      !bias_ok(bias, w.size(0), dev) || !trainable(x.numel() / x.size(-1), w.size(0), x.size(-1)) ||
      (res && (!bf16(*res, dev) || res->dim() != x.dim() || res->size(-1) != w.size(0) ||
               res->sizes().slice(0, x.dim() - 1) != x.sizes().slice(0, x.dim() - 1))))
    return py::none();
  at::Tensor y;
  {
    NoGil no_gil;
    if (records({&ox, &ow, &bias, &res})) y = LinearNode::apply(x, w, bias, res, (int64_t)act);
    else y = linear_run(x, w, bias, act, res, false, vp(stream)).y;
  }
  return py::cast(y);
}

// (x_new, act(h w^T + bias)) for the norm of x + a (x_new None without a), x [..., K] bf16
py::object norm_linear_rows(const at::Tensor &x, const at::Tensor &wn, double eps, const opt &a, const at::Tensor &w,
                            const opt &bias, int act, int dev, handle, handle stream) {
  NormIn in;
  const opt ox = x, own = wn, ow = w, none;
  if (!norm_ok(x, wn, a, none, none, none, dev, in) || !rows_weight_ok(w, x.size(-1), dev) ||
      !bias_ok(bias, w.size(0), dev) || !trainable(x.numel() / x.size(-1), w.size(0), x.size(-1)))
    return py::none();
  at::Tensor xn, y;
  {
    NoGil no_gil;
    if (records({&ox, &own, &a, &ow, &bias})) {
      variable_list o = NormLinearNode::apply(x, wn, w, a, bias, eps, (int64_t)act);
      y = o.back();
      if (a) xn = o[0];
    } else {
      const auto [n, o] = norm_linear_run(x, wn, eps, a, in, w, bias, act, false, false, vp(stream));
      y = o.y;
      if (a) xn = n.xn;
    }
  }
  return py::make_tuple(or_none(xn), y);
}

// The forward calls on a weight that is cast already (wq [N, K] e4m3, sw [N]), each one call: one token's linear 8.7 us instead of
// 15.1 with the cast and the GEMM called apart.
bool served_ok(const at::Tensor &x, const at::Tensor &wq, const at::Tensor &sw, const opt &bias, int act, int dev) {
  return operand_rows(wq, dev) && x.dim() >= 1 && x.numel() >= 1 && x.size(-1) == wq.size(1) && wq.size(0) >= 16 &&
         wq.size(0) % (act == GPIC_ACT_SWIGLU ? 32 : 16) == 0 && scales_ok(sw, wq.size(0), dev) && bias_ok(bias, wq.size(0), dev);
}
at::Tensor served_out(const at::Tensor &x, const at::Tensor &wq, int act) {
  std::vector<int64_t> size = x.sizes().vec();
  size.back() = act == GPIC_ACT_SWIGLU ? wq.size(0) / 2 : wq.size(0);
  return make(x, size, at::kBFloat16);
}

// residual + gate act(x w^T + bias), x [..., K] bf16
py::object linear_served(const at::Tensor &x, const at::Tensor &wq, const at::Tensor &sw, const opt &bias, int act,
                         const opt &res, const opt &gate, int dev, handle, handle stream) {
  const opt ox = x, owq = wq, osw = sw;
  if (!served_ok(x, wq, sw, bias, act, dev) || !bf16(x, dev) || !row_castable(x, dev) ||
      records({&ox, &owq, &osw, &bias, &res, &gate}))
    return py::none();
  const int64_t K = x.size(-1), M = x.numel() / K, N = wq.size(0), No = act == GPIC_ACT_SWIGLU ? N / 2 : N;
  GemmIn g{nullptr, ptr<uint8_t>(wq), nullptr, ptr<float>(sw), M, N, K, &bias, act, u16(res)};
  if ((res && (!bf16(*res, dev) || res->dim() != x.dim() || res->size(-1) != No ||
               res->sizes().slice(0, x.dim() - 1) != x.sizes().slice(0, x.dim() - 1))) ||
      !mod_ok(gate, No, x.dim() > 2 ? x.size(0) : 0, M, dev, g.gate))
    return py::none();
  at::Tensor y;
  {
    NoGil no_gil;
    y = served_out(x, wq, act);
    Arena m;
    const size_t bytes = gpic_fp8_gemm_workspace_bytes(M, N, K), q = m.add(M * K), s = m.add(4 * M), ws = m.add(bytes);
    m.make_like(x);
    check(gpic_fp8_tcast_rows(x.data_ptr(), GPIC_DTYPE_BF16, K, M, K, m.at<uint8_t>(q), m.at<float>(s), nullptr, 0, 0, 0, nullptr,
                              nullptr, vp(stream)),
          "gpic_fp8_tcast_rows");
    g.a = m.at<uint8_t>(q);
    g.sa = m.at<float>(s);
    gemm_rows_call(g, ptr<uint16_t>(y), nullptr, m.at<uint8_t>(ws), bytes, vp(stream));
  }
  return py::cast(y);
}

// (x_new, act(h w^T + bias)) for rmsnorm_rows' x_new and h (x_new None without a)
py::object norm_linear_served(const at::Tensor &x, const at::Tensor &wn, double eps, const opt &a, const opt &gate,
                              const opt &shift, const opt &scale, const at::Tensor &wq, const at::Tensor &sw, const opt &bias,
                              int act, int dev, handle, handle stream) {
  NormIn in;
  const opt ox = x, own = wn, owq = wq, osw = sw;
  if (!norm_ok(x, wn, a, gate, shift, scale, dev, in) || !served_ok(x, wq, sw, bias, act, dev) ||
      records({&ox, &own, &a, &gate, &shift, &scale, &owq, &osw, &bias}))
    return py::none();
  const int64_t K = x.size(-1), M = x.numel() / K, N = wq.size(0);
  at::Tensor y;
  NormOut n;
  {
    NoGil no_gil;
    y = served_out(x, wq, act);
    Arena m;
    const size_t bytes = gpic_fp8_gemm_workspace_bytes(M, N, K), q = m.add(M * K), s = m.add(4 * M), ws = m.add(bytes);
    m.make_like(x);
    n = norm_run(x, wn, eps, a, in, false, m.at<uint8_t>(q), m.at<float>(s), nullptr, nullptr, nullptr, vp(stream));
    const GemmIn g{m.at<uint8_t>(q), ptr<uint8_t>(wq), m.at<float>(s), ptr<float>(sw), M, N, K, &bias, act};
    gemm_rows_call(g, ptr<uint16_t>(y), nullptr, m.at<uint8_t>(ws), bytes, vp(stream));
  }
  return py::make_tuple(a ? py::cast(n.xn) : py::none(), y);
}

// ------------------------------------------------------------------------------------------- layer norm

int dtype_code3(const at::Tensor &t) { return t.scalar_type() == at::kHalf ? GPIC_DTYPE_F16 : dtype_code(t); }
bool float3(at::ScalarType t) { return t == at::kBFloat16 || t == at::kFloat || t == at::kHalf; }
// A weight or bias of n elements, or none
bool vector3_ok(const opt &t, int64_t n, int dev) {
  return !t || (float3(t->scalar_type()) && plain(*t, dev) && t->dim() == 1 && t->size(0) == n);
}
bool layer_norm_ok(const at::Tensor &x, const opt &w, const opt &b, const opt &a, bool bf16_only, int dev) {
  if (x.dim() < 1 || (bf16_only ? x.scalar_type() != at::kBFloat16 : !float3(x.scalar_type())) || !plain(x, dev)) return false;
  const int64_t C = x.size(-1);
  return C > 0 && C % 8 == 0 && C <= kRowsMaxNorm && x.numel() > 0 && vector3_ok(w, C, dev) && vector3_ok(b, C, dev) &&
         (!a || (a->scalar_type() == x.scalar_type() && a->sizes() == x.sizes() && plain(*a, dev)));
}
struct LayerNormOut {
  at::Tensor xn, h, mean, rstd, q, s;
};
LayerNormOut layer_norm_run(const at::Tensor &x, const opt &w, const opt &b, double eps, const opt &a, bool want_h, bool stats,
                            bool rows, void *stream) {
  const int64_t C = x.size(-1), M = x.numel() / C;
  LayerNormOut o;
  o.xn = a ? make(x, x.sizes(), x.scalar_type()) : none_of(x, x.scalar_type());
  o.h = want_h ? make(x, x.sizes(), x.scalar_type()) : none_of(x, x.scalar_type());
  if (stats) o.mean = make(x, {M}, at::kFloat), o.rstd = make(x, {M}, at::kFloat);
  if (rows) o.q = make(x, x.sizes(), kE4), o.s = make(x, {M}, at::kFloat);
  check(gpic_fp8_layer_norm(x.data_ptr(), dtype_code3(x), C, a ? a->data_ptr() : nullptr, C, w ? w->data_ptr() : nullptr,
                            w ? dtype_code3(*w) : 0, b ? b->data_ptr() : nullptr, b ? dtype_code3(*b) : 0, M, C, (float)eps,
                            a ? o.xn.data_ptr() : nullptr, want_h ? o.h.data_ptr() : nullptr,
                            stats ? ptr<float>(o.mean) : nullptr, stats ? ptr<float>(o.rstd) : nullptr,
                            rows ? ptr<uint8_t>(o.q) : nullptr, rows ? ptr<float>(o.s) : nullptr, stream),
        "gpic_fp8_layer_norm");
  return o;
}

// (x_new, h, mean, rstd), the last two empty unless stats; for the op and the autograd Function, which have looked whether a
// gradient is recorded
py::object layer_norm(const at::Tensor &x, const opt &w, const opt &b, double eps, const opt &a, bool stats, int dev, handle,
                      handle stream) {
  if (!layer_norm_ok(x, w, b, a, false, dev)) return py::none();
  LayerNormOut o;
  {
    NoGil no_gil;
    o = layer_norm_run(x, w, b, eps, a, true, stats, false, vp(stream));
    if (!stats) o.mean = none_of(x, at::kFloat), o.rstd = none_of(x, at::kFloat);
  }
  return py::make_tuple(o.xn, o.h, o.mean, o.rstd);
}

py::object layer_norm_rows(const at::Tensor &x, const opt &w, const opt &b, double eps, const opt &a, bool want_h, int dev, handle,
                           handle stream) {
  const opt ox = x;
  if (!layer_norm_ok(x, w, b, a, true, dev) || records({&ox, &w, &b, &a})) return py::none();
  LayerNormOut o;
  {
    NoGil no_gil;
    o = layer_norm_run(x, w, b, eps, a, want_h, false, true, vp(stream));
  }
  return py::make_tuple(o.xn, o.h, o.q, o.s);
}

struct LayerNormGrads {
  at::Tensor dx, dw, db;
};
LayerNormGrads layer_norm_bwd_run(const at::Tensor &dh, const opt &dxn, const at::Tensor &xs, const opt &w, const at::Tensor &mean,
                                  const at::Tensor &rstd, const std::optional<at::ScalarType> &bias_dtype, void *stream) {
  const int64_t C = xs.size(-1), M = xs.numel() / C;
  LayerNormGrads o;
  o.dx = make(xs, xs.sizes(), xs.scalar_type());
  if (w) o.dw = make(xs, {C}, w->scalar_type());
  if (bias_dtype) o.db = make(xs, {C}, *bias_dtype);
  const size_t bytes = gpic_fp8_layer_norm_bwd_workspace_bytes(M, C);
  const at::Tensor ws = make(xs, {(int64_t)bytes}, at::kByte);
  check(gpic_fp8_layer_norm_bwd(dh.data_ptr(), dxn ? dxn->data_ptr() : nullptr, xs.data_ptr(), dtype_code3(xs),
                                w ? w->data_ptr() : nullptr, w ? dtype_code3(*w) : 0, ptr<float>(mean), ptr<float>(rstd), M, C,
                                o.dx.data_ptr(), w ? o.dw.data_ptr() : nullptr, w ? dtype_code3(o.dw) : 0,
                                bias_dtype ? o.db.data_ptr() : nullptr, bias_dtype ? dtype_code3(o.db) : 0, ws.data_ptr(), bytes,
                                stream),
        "gpic_fp8_layer_norm_bwd");
  return o;
}
bool layer_norm_bwd_ok(const at::Tensor &dh, const opt &dxn, const at::Tensor &xs, const opt &w, const at::Tensor &mean,
                       const at::Tensor &rstd, int dev) {
  if (!layer_norm_ok(xs, w, std::nullopt, dxn, false, dev) || dh.scalar_type() != xs.scalar_type() || dh.sizes() != xs.sizes() ||
      !plain(dh, dev))
    return false;
  const int64_t M = xs.numel() / xs.size(-1);
  return scales_ok(mean, M, dev) && scales_ok(rstd, M, dev);
}

py::object layer_norm_bwd(const at::Tensor &dh, const opt &dxn, const at::Tensor &xs, const opt &w, const at::Tensor &mean,
                          const at::Tensor &rstd, const std::optional<at::ScalarType> &bias_dtype, int dev, handle,
                          handle stream) {
  const opt odh = dh, oxs = xs, om = mean, ors = rstd;
  if (!layer_norm_bwd_ok(dh, dxn, xs, w, mean, rstd, dev) || (bias_dtype && !float3(*bias_dtype)) ||
      records({&odh, &dxn, &oxs, &w, &om, &ors}))
    return py::none();
  LayerNormGrads o;
  {
    NoGil no_gil;
    o = layer_norm_bwd_run(dh, dxn, xs, w, mean, rstd, bias_dtype, vp(stream));
    if (!w) o.dw = none_of(xs, at::kFloat);
    if (!bias_dtype) o.db = none_of(xs, at::kFloat);
  }
  return py::make_tuple(o.dx, o.dw, o.db);
}

// The autograd Functions of gpic_fp8/layernorm.py and attention.py in their usual form as nodes of the graph, without a Python
// frame on either of the engine's threads. Their gradients would be constants in a backward that is itself recorded: it throws.
void differentiable_once(const char *what) {
  if (c10::GradMode::is_enabled())
    throw std::runtime_error(std::string(what) + " is differentiable once: its backward does not run under create_graph=True");
}
void saved_as_they_were(bool ok, const char *what) {
  if (!ok) throw std::runtime_error(std::string(what) + "'s backward needs the tensors that the forward saved, as they were saved");
}
// An output's gradient of like's type, contiguous, 16-byte aligned.
at::Tensor usual_as(const at::Tensor &g, const at::Tensor &like) {
  at::Tensor t = g.to(like.scalar_type()).contiguous();
  return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) ? t.clone() : t;
}
opt defined_or_none(const at::Tensor &t) { return t.defined() ? opt(t) : std::nullopt; }

struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
  // (x_new, h), or h alone without a
  static variable_list forward(AutogradContext *ctx, const at::Tensor &x, const opt &w, const opt &b, const opt &a, double eps) {
    const LayerNormOut o = layer_norm_run(x, w, b, eps, a, true, true, false, current_stream(x));
    ctx->save_for_backward({a ? o.xn : x, w ? *w : at::Tensor(), o.mean, o.rstd});
    ctx->set_materialize_grads(false);
    ctx->saved_data["parts"] = (int64_t)((w ? 1 : 0) | (a ? 2 : 0) | (b ? 4 + 8 * (int64_t)b->scalar_type() : 0));
    if (a) return {o.xn, o.h};
    return {o.h};
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &out) {
    differentiable_once("layer_norm");
    variable_list g(5);
    const int64_t parts = ctx->saved_data["parts"].toInt();
    const bool has_w = parts & 1, has_a = parts & 2, has_b = parts & 4;
    const at::Tensor &dxn_ = has_a ? out[0] : at::Tensor(), &dh_ = out.back();
    if (!dh_.defined() && !dxn_.defined()) return g;
    const variable_list s = ctx->get_saved_variables();
    const at::Tensor &xs = s[0], &mean = s[2], &rstd = s[3];
    const opt w = defined_or_none(s[1]);
    size_t edge = 1;
    const bool dx = ctx->needs_input_grad(0), dw = has_w && ctx->needs_input_grad(edge++),
               db = has_b && ctx->needs_input_grad(edge++), da = has_a && ctx->needs_input_grad(edge);
    const auto bt = (at::ScalarType)(parts >> 3);
    const opt dxn = dxn_.defined() ? opt(usual_as(dxn_, xs)) : std::nullopt;
    LayerNormGrads o;
    if (!dh_.defined()) {   // (x_new alone was used: its gradient as it is, and zeros that no value of x can spoil)
      o.dx = *dxn;
      if (dw) o.dw = at::zeros({xs.size(-1)}, dxn->options().dtype(w->scalar_type()));
      if (db) o.db = at::zeros({xs.size(-1)}, dxn->options().dtype(bt));
    } else {
      const at::Tensor dh = usual_as(dh_, xs);
      saved_as_they_were(has_w == w.has_value() && layer_norm_bwd_ok(dh, dxn, xs, w, mean, rstd, dh.get_device()), "layer_norm");
      o = layer_norm_bwd_run(dh, dxn, xs, w, mean, rstd, db ? std::optional<at::ScalarType>(bt) : std::nullopt,
                             current_stream(dh));
    }
    if (dx) g[0] = o.dx;
    if (dw) g[1] = o.dw;
    if (db) g[2] = o.db;
    if (da) g[3] = o.dx;
    return g;
  }
};

// The public call: h, or (x_new, h); a node of the graph where it records
py::object layer_norm_call(const at::Tensor &x, const opt &w, const opt &b, double eps, const opt &a, int dev, handle,
                           handle stream) {
  const opt ox = x;
  if (!layer_norm_ok(x, w, b, a, false, dev)) return py::none();
  at::Tensor xn, h;
  {
    NoGil no_gil;
    if (records({&ox, &w, &b, &a})) {
      variable_list o = LayerNormNode::apply(x, w, b, a, eps);
      h = o.back();
      if (a) xn = o[0];
    } else {
      const LayerNormOut o = layer_norm_run(x, w, b, eps, a, true, false, false, vp(stream));
      xn = o.xn, h = o.h;
    }
  }
  if (!a) return py::cast(h);
  return py::make_tuple(xn, h);
}

// ------------------------------------------------------------------------------------------- attention

// [B, H, N, D] as the kernels read it, and its strides (0 for an extent of one)
bool heads_ok(const at::Tensor &t, at::ScalarType ty, int dev, int64_t (&s)[3]) {
  if (t.dim() != 4 || t.scalar_type() != ty || !t.is_cuda() || t.get_device() != dev || !has_memory(t) ||
      t.layout() != at::kStrided || t.numel() == 0 || t.stride(3) != 1 || (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u))
    return false;
  for (int i = 0; i < 3; i++) {
    s[i] = t.size(i) > 1 ? t.stride(i) : 0;
    if (s[i] % 8) return false;
  }
  return true;
}
struct AttnIn {
  int64_t B, H, Hk, N, L, D, qs[3], ks[3], vs[3], ldm = 0;
  const int *lens = nullptr;
  const uint8_t *mask = nullptr;
  int dtype;
};
bool attn_ok(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const opt &lens, const opt &mask, double scale, int dev,
             AttnIn &in) {
  const at::ScalarType ty = q.scalar_type();
  if ((ty != at::kBFloat16 && ty != at::kHalf) || !heads_ok(q, ty, dev, in.qs) || !heads_ok(k, ty, dev, in.ks) ||
      !heads_ok(v, ty, dev, in.vs) || k.sizes() != v.sizes() || q.size(0) != k.size(0) || q.size(3) != k.size(3))
    return false;
  in.B = q.size(0), in.H = q.size(1), in.N = q.size(2), in.D = q.size(3), in.Hk = k.size(1), in.L = k.size(2);
  in.dtype = ty == at::kHalf ? GPIC_DTYPE_F16 : GPIC_DTYPE_BF16;
  if (in.D > 128 || in.D % 8 || in.H % in.Hk || !(scale > 0.0) || !((float)scale < INFINITY)) return false;
  if (lens) {
    if (lens->scalar_type() != at::kInt || lens->dim() != 1 || lens->size(0) != in.B || !lens->is_cuda() ||
        lens->get_device() != dev || !has_memory(*lens) || !lens->is_contiguous())
      return false;
    in.lens = ptr<int>(*lens);
  }
  if (mask) {
    if (mask->scalar_type() != at::kBool || mask->dim() != 2 || mask->size(0) != in.B || mask->size(1) != in.L || !mask->is_cuda() ||
        mask->get_device() != dev || !has_memory(*mask) || mask->layout() != at::kStrided || mask->stride(1) != 1 ||
        mask->stride(0) < 0)
      return false;
    in.mask = static_cast<const uint8_t *>(mask->data_ptr());
    in.ldm = mask->stride(0);
  }
  return true;
}
// [B, H, N, D], [B, N, H, D] in memory: a view of a new tensor, as the general form makes it
at::Tensor make_heads(const at::Tensor &like, int64_t B, int64_t H, int64_t N, int64_t D, int64_t (&s)[3]) {
  s[0] = N * H * D, s[1] = D, s[2] = H * D;
  return make(like, {B, N, H, D}, like.scalar_type()).transpose(1, 2);
}
at::Tensor attn_run(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const AttnIn &in, double scale, float *lse,
                    void *stream) {
  int64_t os[3];
  at::Tensor o = make_heads(q, in.B, in.H, in.N, in.D, os);
  const size_t bytes = gpic_fp8_attention_workspace_bytes(in.B, in.H, in.Hk, in.N, in.L, in.D);
  at::Tensor ws;
  if (bytes) ws = make(q, {(int64_t)bytes}, at::kByte);
  check(gpic_fp8_attention(ptr<uint16_t>(q), in.qs, ptr<uint16_t>(k), in.ks, ptr<uint16_t>(v), in.vs, in.dtype, in.lens, in.mask,
                           in.ldm, in.B, in.H, in.Hk, in.N, in.L, in.D, (float)scale, ptr<uint16_t>(o), os, lse,
                           bytes ? ws.data_ptr() : nullptr, bytes, stream),
        "gpic_fp8_attention");
  return o;
}

// (o, lse, empty unless asked for); for the op and the autograd Function, which have looked whether a gradient is recorded
py::object attention(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const opt &lens, const opt &mask, double scale,
                     bool want_lse, int dev, handle, handle stream) {
  AttnIn in;
  const opt oq = q, ok = k, ov = v;
  if (!attn_ok(q, k, v, lens, mask, scale, dev, in) || records({&oq, &ok, &ov})) return py::none();
  at::Tensor o, lse;
  {
    NoGil no_gil;
    at::AutoDispatchBelowADInplaceOrView below;
    lse = want_lse ? make(q, {in.B, in.H, in.N}, at::kFloat) : none_of(q, at::kFloat);
    o = attn_run(q, k, v, in, scale, want_lse ? ptr<float>(lse) : nullptr, vp(stream));
  }
  return py::make_tuple(o, lse);
}

struct AttnGrads {
  at::Tensor dq, dk, dv;
};
bool attn_bwd_ok(const at::Tensor &dout, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &o,
                 const at::Tensor &lse, const opt &lens, const opt &mask, double scale, int dev, AttnIn &in, int64_t (&ds)[3],
                 int64_t (&os)[3]) {
  const at::ScalarType ty = q.scalar_type();
  return attn_ok(q, k, v, lens, mask, scale, dev, in) && heads_ok(dout, ty, dev, ds) && heads_ok(o, ty, dev, os) &&
         dout.sizes() == q.sizes() && o.sizes() == q.sizes() && lse.dim() == 3 && lse.scalar_type() == at::kFloat &&
         plain(lse, dev) && lse.size(0) == in.B && lse.size(1) == in.H && lse.size(2) == in.N;
}
AttnGrads attn_bwd_run(const at::Tensor &dout, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &o,
                       const at::Tensor &lse, double scale, bool want_kv, const AttnIn &in, const int64_t (&ds)[3],
                       const int64_t (&os)[3], void *stream) {
  int64_t dqs[3], dks[3], dvs[3];
  AttnGrads r;
  r.dq = make_heads(q, in.B, in.H, in.N, in.D, dqs);
  if (want_kv) {
    r.dk = make_heads(q, in.B, in.Hk, in.L, in.D, dks);
    r.dv = make_heads(q, in.B, in.Hk, in.L, in.D, dvs);
  }
  const size_t bytes = gpic_fp8_attention_bwd_workspace_bytes(in.B, in.H, in.Hk, in.N, in.L, in.D);
  const at::Tensor ws = make(q, {std::max<int64_t>((int64_t)bytes, 16)}, at::kByte);
  check(gpic_fp8_attention_bwd(ptr<uint16_t>(dout), ds, ptr<uint16_t>(q), in.qs, ptr<uint16_t>(k), in.ks, ptr<uint16_t>(v), in.vs,
                               ptr<uint16_t>(o), os, ptr<float>(lse), in.dtype, in.lens, in.mask, in.ldm, in.B, in.H, in.Hk, in.N,
                               in.L, in.D, (float)scale, ptr<uint16_t>(r.dq), dqs, want_kv ? ptr<uint16_t>(r.dk) : nullptr, dks,
                               want_kv ? ptr<uint16_t>(r.dv) : nullptr, dvs, ws.data_ptr(), bytes, stream),
        "gpic_fp8_attention_bwd");
  return r;
}

py::object attention_bwd(const at::Tensor &dout, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &o,
                         const at::Tensor &lse, const opt &lens, const opt &mask, double scale, bool want_kv, int dev, handle,
                         handle stream) {
  AttnIn in;
  int64_t ds[3], os[3];
  const opt od = dout, oq = q, ok = k, ov = v, oo = o, ol = lse;
  if (!attn_bwd_ok(dout, q, k, v, o, lse, lens, mask, scale, dev, in, ds, os) || records({&od, &oq, &ok, &ov, &oo, &ol}))
    return py::none();
  AttnGrads r;
  {
    NoGil no_gil;
    at::AutoDispatchBelowADInplaceOrView below;
    r = attn_bwd_run(dout, q, k, v, o, lse, scale, want_kv, in, ds, os, vp(stream));
    if (!want_kv) r.dk = none_of(q, q.scalar_type()), r.dv = none_of(q, q.scalar_type());
  }
  return py::make_tuple(r.dq, r.dk, r.dv);
}

struct AttentionNode : torch::autograd::Function<AttentionNode> {
  static at::Tensor forward(AutogradContext *ctx, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const opt &lens,
                            const opt &mask, double scale) {
    at::AutoDispatchBelowADInplaceOrView below;   // (o is a tensor of its own, not a view)
    AttnIn in;
    saved_as_they_were(attn_ok(q, k, v, lens, mask, scale, q.get_device(), in), "cross_attention");
    const at::Tensor lse = make(q, {in.B, in.H, in.N}, at::kFloat);
    const at::Tensor o = attn_run(q, k, v, in, scale, ptr<float>(lse), current_stream(q));
    ctx->save_for_backward({q, k, v, o, lse, lens ? *lens : at::Tensor(), mask ? *mask : at::Tensor()});
    ctx->set_materialize_grads(false);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["keys"] = (int64_t)((lens ? 1 : 0) | (mask ? 2 : 0));
    return o;
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &out) {
    differentiable_once("cross_attention");
    variable_list g(6);
    if (!out[0].defined()) return g;
    const variable_list s = ctx->get_saved_variables();
    const opt lens = defined_or_none(s[5]), mask = defined_or_none(s[6]);
    const double scale = ctx->saved_data["scale"].toDouble();
    const int64_t keys = ctx->saved_data["keys"].toInt();
    at::AutoDispatchBelowADInplaceOrView below;
    at::Tensor dout = out[0].to(s[0].scalar_type());
    AttnIn in;
    int64_t ds[3], os[3];
    const int dev = dout.get_device();
    if (!heads_ok(dout, dout.scalar_type(), dev, ds)) dout = usual_as(dout.transpose(1, 2), dout).transpose(1, 2);
    saved_as_they_were(((keys & 1) != 0) == lens.has_value() && ((keys & 2) != 0) == mask.has_value() &&
                           attn_bwd_ok(dout, s[0], s[1], s[2], s[3], s[4], lens, mask, scale, dev, in, ds, os),
                       "cross_attention");
    const bool nk = ctx->needs_input_grad(1), nv = ctx->needs_input_grad(2);
    AttnGrads r = attn_bwd_run(dout, s[0], s[1], s[2], s[3], s[4], scale, nk || nv, in, ds, os, current_stream(dout));
    if (ctx->needs_input_grad(0)) g[0] = r.dq;
    if (nk) g[1] = r.dk;
    if (nv) g[2] = r.dv;
    return g;
  }
};

// The public call; a node of the graph where it records
py::object attention_call(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const opt &lens, const opt &mask,
                          double scale, int dev, handle, handle stream) {
  AttnIn in;
  const opt oq = q, ok = k, ov = v;
  if (!attn_ok(q, k, v, lens, mask, scale, dev, in)) return py::none();
  at::Tensor o;
  {
    NoGil no_gil;
    if (records({&oq, &ok, &ov})) {
      o = AttentionNode::apply(q, k, v, lens, mask, scale);
    } else {
      at::AutoDispatchBelowADInplaceOrView below;
      o = attn_run(q, k, v, in, scale, nullptr, vp(stream));
    }
  }
  return py::cast(o);
}

// ------------------------------------------------------------------------------------------- adapters

py::object lora_rows(const at::Tensor &y, const at::Tensor &x, const at::Tensor &A, const at::Tensor &B, const at::Tensor &ids,
                     const opt &scale, int dev, handle, handle stream) {
  const at::ScalarType ty = y.scalar_type();
  const opt oy = y, ox = x, oA = A, oB = B;
  if ((ty != at::kBFloat16 && ty != at::kHalf) || x.scalar_type() != ty || A.scalar_type() != ty || B.scalar_type() != ty ||
      y.dim() < 2 || x.dim() != y.dim() || A.dim() != 3 || B.dim() != 3 || !plain(y, dev) || !plain(x, dev) || !plain(A, dev) ||
      !plain(B, dev) || !plain(ids, dev) || (ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong))
    return py::none();
  const int64_t N = y.size(-1), K = x.size(-1), n = A.size(0), R = A.size(1);
  if (N <= 0 || K <= 0 || n <= 0 || R <= 0 || N % 8 || K % 8 || R % 8 || R > 128 || A.size(2) != K || B.size(0) != n ||
      B.size(1) != N || B.size(2) != R || !scales_ok(scale, n, dev))
    return py::none();
  for (int64_t i = 0; i + 1 < y.dim(); i++)
    if (x.size(i) != y.size(i)) return py::none();
  const int64_t M = x.numel() / K;
  if (M < 1 || (ids.sizes() != x.sizes().slice(0, x.dim() - 1) && !(ids.dim() == 1 && ids.size(0) == x.size(0))) ||
      records({&oy, &ox, &oA, &oB, &scale}))
    return py::none();
  at::Tensor out;
  {
    NoGil no_gil;
    out = make(y, y.sizes(), ty);
    const size_t bytes = gpic_fp8_lora_rows_workspace_bytes(M, N, K, R, n);
    const at::Tensor ws = make(y, {(int64_t)bytes}, at::kByte);
    check(gpic_fp8_lora_rows(ptr<uint16_t>(y), N, ptr<uint16_t>(x), K, ptr<uint16_t>(A), ptr<uint16_t>(B),
                             scale ? ptr<float>(*scale) : nullptr, ids.data_ptr(), ids.scalar_type() == at::kLong,
                             M / ids.numel(), ty == at::kHalf ? GPIC_DTYPE_F16 : GPIC_DTYPE_BF16, M, N, K, R, n, ptr<uint16_t>(out),
                             ws.data_ptr(), bytes, vp(stream)),
          "gpic_fp8_lora_rows");
  }
  return py::cast(out);
}

}  // namespace

PYBIND11_MODULE(_gpic_host, m) {   // (wrapped: torch's own errors, out of memory among them, stay what they are)
  m.def("casts", torch::wrap_pybind_function(&casts));
  m.def("gemm", torch::wrap_pybind_function(&gemm));
  m.def("wgrad", torch::wrap_pybind_function(&wgrad));
  m.def("linear_fwd", torch::wrap_pybind_function(&linear_fwd));
  m.def("linear_bwd", torch::wrap_pybind_function(&linear_bwd));
  m.def("cast_rows", torch::wrap_pybind_function(&cast_rows));
  m.def("norm_rows", torch::wrap_pybind_function(&norm_rows));
  m.def("norm_rows_bwd", torch::wrap_pybind_function(&norm_rows_bwd));
  m.def("gemm_rows", torch::wrap_pybind_function(&gemm_rows));
  m.def("layer_norm", torch::wrap_pybind_function(&layer_norm));
  m.def("layer_norm_call", torch::wrap_pybind_function(&layer_norm_call));
  m.def("layer_norm_rows", torch::wrap_pybind_function(&layer_norm_rows));
  m.def("layer_norm_bwd", torch::wrap_pybind_function(&layer_norm_bwd));
  m.def("attention", torch::wrap_pybind_function(&attention));
  m.def("attention_call", torch::wrap_pybind_function(&attention_call));
  m.def("attention_bwd", torch::wrap_pybind_function(&attention_bwd));
  m.def("lora_rows", torch::wrap_pybind_function(&lora_rows));
  m.def("linear_rows_bwd", torch::wrap_pybind_function(&linear_rows_bwd));
  m.def("norm_linear_rows_fwd", torch::wrap_pybind_function(&norm_linear_rows_fwd));
  m.def("linear_rows", torch::wrap_pybind_function(&linear_rows));
  m.def("norm_linear_rows", torch::wrap_pybind_function(&norm_linear_rows));
  m.def("linear_served", torch::wrap_pybind_function(&linear_served));
  m.def("norm_linear_served", torch::wrap_pybind_function(&norm_linear_served));
}
