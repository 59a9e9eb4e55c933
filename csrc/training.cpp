// Python binding of the transformer block's training kernels.
//
// Host-side glue only: the checks of the arguments (TypeError and ValueError
// in Python, the same as kfac_amd.ops raises on the CPU), allocation,
// launches on the current stream of the tensors' device. Small calls are
// bound by the host, so allocation goes past the dispatcher.

#include "training.h"

#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <cstdlib>
#include <cstring>
#include <tuple>

namespace {

using torch::Tensor;
using OptTensor = std::optional<Tensor>;
using Borrowed = c10::MaybeOwned<Tensor>;

#define CHECK_OK(expr)                                                       \
  do {                                                                       \
    hipError_t _e = (expr);                                                  \
    TORCH_CHECK(_e == hipSuccess, "HIP error: ", hipGetErrorString(_e));     \
  } while (0)

hipStream_t stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

Tensor empty(
    at::IntArrayRef size,
    torch::ScalarType type,
    const Tensor& like) {
  return at::detail::empty_cuda(size, type, like.device(), std::nullopt);
}

Tensor zeros(
    at::IntArrayRef size,
    torch::ScalarType type,
    const Tensor& like) {
  return empty(size, type, like).zero_();
}

bool is_float(torch::ScalarType st) {
  return st == torch::kFloat32 || st == torch::kBFloat16 ||
      st == torch::kFloat16;
}

int type_of(torch::ScalarType st) {
  return st == torch::kFloat32 ? kfac::kF32
      : st == torch::kBFloat16 ? kfac::kBF16
                               : kfac::kF16;
}

// Calls fn with a value of the C++ type; the type has been checked.
template <typename Fn>
void by_type(torch::ScalarType st, Fn fn) {
  if (st == torch::kFloat32) {
    fn(float());
  } else if (st == torch::kBFloat16) {
    fn(__hip_bfloat16());
  } else {
    fn(__half());
  }
}

struct Shape {
  long R;
  int D;
  long blocks;
};

Shape shape_of(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(
      t.dim() >= 1 && t.size(-1) >= 1, name,
      " must have rows of one value or more, got shape ", t.sizes());
  const long D = t.size(-1);
  TORCH_CHECK_VALUE(D < (1L << 30), name, " has rows of 2^30 values or more");
  return {t.numel() / D, (int)D, (D + kfac::kBlock8 - 1) / kfac::kBlock8};
}

void check_float(torch::ScalarType st, const char* name) {
  TORCH_CHECK_TYPE(
      is_float(st), name, " must be float32, bfloat16 or float16, got ", st);
}

Shape check_rows(const Tensor& t, const char* name) {
  check_float(t.scalar_type(), name);
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a GPU tensor");
  return shape_of(t, name);
}

void check_like(const Tensor& t, const Tensor& like, const char* names) {
  TORCH_CHECK_VALUE(
      t.device() == like.device() && t.sizes() == like.sizes(), names,
      " must have the same shape and device, got ", t.sizes(), " on ",
      t.device(), " and ", like.sizes(), " on ", like.device());
}

Shape check_packed(const Tensor& codes, const Tensor& exps) {
  TORCH_CHECK_TYPE(
      codes.scalar_type() == torch::kInt8 &&
          exps.scalar_type() == torch::kUInt8,
      "a Packed8 holds int8 codes and uint8 exponents, got ",
      codes.scalar_type(), " and ", exps.scalar_type());
  TORCH_CHECK_VALUE(codes.is_cuda(), "codes must be a GPU tensor");
  const Shape s = shape_of(codes, "codes");
  TORCH_CHECK_VALUE(
      exps.device() == codes.device() && exps.dim() == codes.dim() &&
          exps.size(-1) == s.blocks &&
          exps.sizes().slice(0, exps.dim() - 1) ==
              codes.sizes().slice(0, codes.dim() - 1),
      "codes of shape ", codes.sizes(), " do not go with exponents of shape ",
      exps.sizes());
  return s;
}

// The 8 bit form of a tensor like `like`: its codes, its exponents.
std::tuple<Tensor, Tensor> empty_packed(const Tensor& like, long blocks) {
  at::DimVector size(like.sizes());
  auto codes = empty(size, torch::kInt8, like);
  size.back() = blocks;
  return {std::move(codes), empty(size, torch::kUInt8, like)};
}

// The 8 bit forms of an input and an output that a call asks for, null where
// it does not; their tensors are appended to `out`.
struct Packs {
  int8_t* codes[2] = {};
  uint8_t* exps[2] = {};

  Packs(
      const Tensor& like,
      long blocks,
      bool input,
      bool output,
      std::vector<Tensor>& out) {
    for (int i = 0; i < 2; ++i) {
      if (!(i ? output : input)) continue;
      auto [c, e] = empty_packed(like, blocks);
      codes[i] = (int8_t*)c.data_ptr();
      exps[i] = (uint8_t*)e.data_ptr();
      out.push_back(std::move(c));
      out.push_back(std::move(e));
    }
  }
};

std::tuple<Tensor, Tensor> pack8(const Tensor& x) {
  const Shape s = check_rows(x, "x");
  const c10::DeviceGuard guard(x.device());
  const Borrowed xc = x.expect_contiguous();
  auto packed = empty_packed(x, s.blocks);
  if (s.R > 0) {
    by_type(x.scalar_type(), [&](auto t) {
      using T = decltype(t);
      CHECK_OK(kfac::pack8_t<T>(
          stream_of(x), (const T*)xc->const_data_ptr(),
          (int8_t*)std::get<0>(packed).data_ptr(),
          (uint8_t*)std::get<1>(packed).data_ptr(), s.R, s.D));
    });
  }
  return packed;
}

Tensor unpack8(
    const Tensor& codes,
    const Tensor& exps,
    torch::ScalarType dtype) {
  const Shape s = check_packed(codes, exps);
  check_float(dtype, "dtype");
  const c10::DeviceGuard guard(codes.device());
  const Borrowed cc = codes.expect_contiguous(), ec = exps.expect_contiguous();
  auto out = empty(codes.sizes(), dtype, codes);
  if (s.R > 0) {
    by_type(dtype, [&](auto t) {
      using T = decltype(t);
      CHECK_OK(kfac::unpack8_t<T>(
          stream_of(codes), (const int8_t*)cc->const_data_ptr(),
          (const uint8_t*)ec->const_data_ptr(), (T*)out.data_ptr(), s.R,
          s.D));
    });
  }
  return out;
}

// (y[, codes and exponents of x][, of y])
std::vector<Tensor> gelu8_forward(
    const Tensor& x,
    bool tanh,
    bool pack_input,
    bool pack_output) {
  const Shape s = check_rows(x, "x");
  const c10::DeviceGuard guard(x.device());
  const Borrowed xc = x.expect_contiguous();
  std::vector<Tensor> out{empty(x.sizes(), x.scalar_type(), x)};
  const Packs packs(x, s.blocks, pack_input, pack_output, out);
  if (s.R > 0) {
    by_type(x.scalar_type(), [&](auto t) {
      using T = decltype(t);
      CHECK_OK(kfac::gelu8_fwd_t<T>(
          stream_of(x), (const T*)xc->const_data_ptr(),
          (T*)out[0].data_ptr(), packs.codes[0], packs.exps[0],
          packs.codes[1], packs.exps[1], s.R, s.D, tanh));
    });
  }
  return out;
}

Tensor gelu8_backward(
    const Tensor& dy,
    const Tensor& codes,
    const Tensor& exps,
    bool tanh) {
  check_rows(dy, "dy");
  const Shape s = check_packed(codes, exps);
  check_like(dy, codes, "dy and the packed input");
  const c10::DeviceGuard guard(dy.device());
  const Borrowed dc = dy.expect_contiguous();
  const Borrowed cc = codes.expect_contiguous(), ec = exps.expect_contiguous();
  auto dx = empty(dy.sizes(), dy.scalar_type(), dy);
  if (s.R > 0) {
    by_type(dy.scalar_type(), [&](auto t) {
      using T = decltype(t);
      CHECK_OK(kfac::gelu8_bwd_t<T>(
          stream_of(dy), (const T*)dc->const_data_ptr(),
          (const int8_t*)cc->const_data_ptr(),
          (const uint8_t*)ec->const_data_ptr(), (T*)dx.data_ptr(), s.R, s.D,
          tanh));
    });
  }
  return dx;
}

// The types of a norm's inner (x, dx) and outer (y, dy) tensors: the same,
// or one of them fp32.
void check_types(torch::ScalarType inner, torch::ScalarType outer) {
  TORCH_CHECK_TYPE(
      is_float(outer) &&
          (inner == outer || inner == torch::kFloat32 ||
           outer == torch::kFloat32),
      "no layer norm from ", inner, " to ", outer,
      ": the types must be the same or one of them float32");
}

template <typename Fn>
void by_types(torch::ScalarType x, torch::ScalarType y, Fn fn) {
  by_type(x, [&](auto tx) {
    using TX = decltype(tx);
    if (x == y) {
      fn(tx, tx);
    } else if constexpr (std::is_same_v<TX, float>) {
      by_type(y, [&](auto ty) { fn(tx, ty); });
    } else {
      fn(tx, float());
    }
  });
}

// A tensor that may be missing: contiguous, with its pointer and type.
struct Param {
  std::optional<Borrowed> held;
  const void* p = nullptr;
  int type = kfac::kF32;

  explicit Param(const OptTensor& t) {
    if (!t) return;
    held.emplace(t->expect_contiguous());
    p = (*held)->const_data_ptr();
    if (is_float(t->scalar_type())) type = type_of(t->scalar_type());
  }
};

void check_param(const OptTensor& t, const char* name, const Tensor& x) {
  if (!t) return;
  check_float(t->scalar_type(), name);
  TORCH_CHECK_VALUE(
      t->dim() == 1 && t->size(0) == x.size(-1) && t->device() == x.device(),
      name, " must have shape (", x.size(-1), ",) on ", x.device(), ", got ",
      t->sizes(), " on ", t->device());
}

// (y, total or x, mean, rstd[, codes, exponents of the input][, of the
// output])
std::vector<Tensor> norm_forward(
    const Tensor& x,
    const OptTensor& r,
    const OptTensor& w,
    const OptTensor& b,
    double eps,
    std::optional<torch::ScalarType> out_dtype,
    bool pack_input,
    bool pack_output) {
  const Shape s = check_rows(x, "x");
  const auto xt = x.scalar_type(), yt = out_dtype.value_or(xt);
  check_types(xt, yt);
  check_param(w, "weight", x);
  check_param(b, "bias", x);
  if (r) {
    check_float(r->scalar_type(), "residual");
    check_like(x, *r, "x and residual");
    TORCH_CHECK_TYPE(
        r->scalar_type() == xt || xt == torch::kFloat32, "a residual of ",
        r->scalar_type(), " does not fit a sum of ", xt);
  }
  const c10::DeviceGuard guard(x.device());
  const Borrowed xc = x.expect_contiguous();
  const Param rp(r), wp(w), bp(b);
  std::vector<Tensor> out;
  out.reserve(8);
  out.push_back(empty(x.sizes(), yt, x));
  out.push_back(r ? empty(x.sizes(), xt, x) : *xc);
  out.push_back(empty({s.R}, torch::kFloat32, x));
  out.push_back(empty({s.R}, torch::kFloat32, x));
  const Packs packs(x, s.blocks, pack_input, pack_output, out);
  if (s.R > 0) {
    by_types(xt, yt, [&](auto tx, auto ty) {
      using TX = decltype(tx);
      using TY = decltype(ty);
      CHECK_OK((kfac::norm_fwd_t<TX, TY>(
          stream_of(x), (const TX*)xc->const_data_ptr(), rp.p, rp.type, wp.p,
          wp.type, bp.p, bp.type, r ? (TX*)out[1].data_ptr() : nullptr,
          (TY*)out[0].data_ptr(), (float*)out[2].data_ptr(),
          (float*)out[3].data_ptr(), packs.codes[0], packs.exps[0],
          packs.codes[1], packs.exps[1], s.R, s.D, (float)eps)));
    });
  }
  return out;
}

// (dx, dweight or None, dbias or None); total or (codes, exps)
std::tuple<Tensor, OptTensor, OptTensor> norm_backward(
    const Tensor& dy,
    const OptTensor& total,
    const OptTensor& codes,
    const OptTensor& exps,
    const Tensor& mean,
    const Tensor& rstd,
    const OptTensor& w,
    bool want_dw,
    bool want_db,
    const OptTensor& dt,
    std::optional<torch::ScalarType> dtype,
    std::optional<torch::ScalarType> bias_dtype) {
  const Shape s = check_rows(dy, "dy");
  auto xt = dy.scalar_type();
  if (total) {
    check_float(total->scalar_type(), "total");
    check_like(dy, *total, "dy and total");
    xt = total->scalar_type();
    TORCH_CHECK_TYPE(
        !dtype || *dtype == xt, "dx has the type of total, ", xt);
  } else {
    TORCH_CHECK_VALUE(codes && exps, "total or its 8 bit form is missing");
    check_packed(*codes, *exps);
    check_like(dy, *codes, "dy and total");
    xt = dtype.value_or(xt);
    check_float(xt, "dtype");
  }
  check_types(xt, dy.scalar_type());
  check_param(w, "weight", dy);
  for (const auto* t : {&mean, &rstd}) {
    TORCH_CHECK_VALUE(
        t->scalar_type() == torch::kFloat32 && t->dim() == 1 &&
            t->size(0) == s.R && t->device() == dy.device(),
        t == &mean ? "mean" : "rstd", " must hold a float32 for each row");
  }
  if (dt) {
    check_like(dy, *dt, "dy and grad_total");
    TORCH_CHECK_TYPE(
        dt->scalar_type() == xt, "grad_total must be ", xt, ", as dx is");
  }
  check_float(bias_dtype.value_or(torch::kFloat32), "bias_dtype");
  const c10::DeviceGuard guard(dy.device());
  const Borrowed dc = dy.expect_contiguous();
  const Borrowed mc = mean.expect_contiguous(), rc = rstd.expect_contiguous();
  const Param xp(total), cp(codes), ep(exps), wp(w), tp(dt);
  auto dx = empty(dy.sizes(), xt, dy);
  const auto wt = w ? w->scalar_type() : torch::kFloat32;
  const auto bt = bias_dtype.value_or(wt);
  OptTensor dw, db;
  want_dw = want_dw && w;
  if (s.R == 0) {
    if (want_dw) dw = zeros({s.D}, wt, dy);
    if (want_db) db = zeros({s.D}, bt, dy);
    return {dx, dw, db};
  }
  if (want_dw) dw = empty({s.D}, wt, dy);
  if (want_db) db = empty({s.D}, bt, dy);
  Tensor partial;
  const long rows = dw || db ? kfac::norm_bwd_partials(s.R, s.D) : 0;
  if (rows > 0) partial = empty({rows * 2 * s.D}, torch::kFloat32, dy);
  by_types(xt, dy.scalar_type(), [&](auto tx, auto ty) {
    using TX = decltype(tx);
    using TY = decltype(ty);
    CHECK_OK((kfac::norm_bwd_t<TX, TY>(
        stream_of(dy), (const TY*)dc->const_data_ptr(), (const TX*)xp.p,
        (const int8_t*)cp.p, (const uint8_t*)ep.p,
        (const float*)mc->const_data_ptr(),
        (const float*)rc->const_data_ptr(), wp.p, wp.type, (const TX*)tp.p,
        (TX*)dx.data_ptr(),
        partial.defined() ? (float*)partial.data_ptr() : nullptr,
        dw ? dw->data_ptr() : nullptr, type_of(wt),
        db ? db->data_ptr() : nullptr, type_of(bt), s.R, s.D)));
  });
  return {std::move(dx), std::move(dw), std::move(db)};
}

// (dW, db or None)
std::tuple<Tensor, OptTensor> weight_grad8(
    const Tensor& g,
    const Tensor& codes,
    const Tensor& exps,
    bool want_bias,
    torch::ScalarType dtype,
    std::optional<torch::ScalarType> bias_dtype) {
  const Shape sg = check_rows(g, "g");
  const Shape sx = check_packed(codes, exps);
  TORCH_CHECK_VALUE(
      g.device() == codes.device() && g.dim() == codes.dim() &&
          g.sizes().slice(0, g.dim() - 1) ==
              codes.sizes().slice(0, codes.dim() - 1),
      "g and the packed input must have the same rows and device, got ",
      g.sizes(), " on ", g.device(), " and ", codes.sizes(), " on ",
      codes.device());
  check_float(dtype, "dtype");
  const auto bt = bias_dtype.value_or(dtype);
  check_float(bt, "bias_dtype");
  const c10::DeviceGuard guard(g.device());
  const Borrowed gc = g.expect_contiguous();
  const Borrowed cc = codes.expect_contiguous(), ec = exps.expect_contiguous();
  const long M = sg.R, N = sg.D, K = sx.D;
  // 32 of these rows are addressed with 32 bits
  TORCH_CHECK_VALUE(
      N < (1L << 27) && K < (1L << 27),
      "a weight gradient takes rows of less than 2^27 values");
  OptTensor db;
  if (M == 0) {
    if (want_bias) db = zeros({N}, bt, g);
    return {zeros({N, K}, dtype, g), db};
  }
  auto dw = empty({N, K}, dtype, g);
  if (want_bias) db = empty({N}, bt, g);
  const auto stream = stream_of(g);
  by_type(g.scalar_type(), [&](auto t) {
    using T = decltype(t);
    const auto plan = kfac::wgrad8_plan<T>(M, sg.D, sx.D);
    const long rows = (long)plan.splits * plan.bias_tiles;
    // a single fp32 sum is the result itself; the others share a workspace
    const bool direct = plan.splits == 1 && dtype == torch::kFloat32;
    const bool bias_direct = rows == 1 && bt == torch::kFloat32;
    const long need = direct ? 0 : plan.splits * N * K;
    const long bias_need = want_bias && !bias_direct ? rows * N : 0;
    Tensor work;
    float* sums = (float*)dw.data_ptr();
    float* bias = want_bias ? (float*)db->data_ptr() : nullptr;
    if (need + bias_need > 0) {
      work = empty({need + bias_need}, torch::kFloat32, g);
      if (need > 0) sums = (float*)work.data_ptr();
      if (bias_need > 0) bias = (float*)work.data_ptr() + need;
    }
    CHECK_OK(kfac::wgrad8_t<T>(
        stream, (const T*)gc->const_data_ptr(),
        (const int8_t*)cc->const_data_ptr(),
        (const uint8_t*)ec->const_data_ptr(), M, sg.D, sx.D, plan, sums,
        bias));
    CHECK_OK(kfac::wgrad8_add(
        stream, sums, plan.splits, N * K, need ? dw.data_ptr() : nullptr,
        type_of(dtype), bias, (int)rows, N,
        bias_need ? db->data_ptr() : nullptr, type_of(bt)));
  });
  return {std::move(dw), std::move(db)};
}

// KFAC_AMD_FORCE_EAGER=1, which may change while a program runs
bool force_eager() {
  const char* v = std::getenv("KFAC_AMD_FORCE_EAGER");
  return v != nullptr && std::strcmp(v, "1") == 0;
}

}  // namespace

void bind_training(pybind11::module& m) {
  m.def("force_eager", &force_eager, "whether the kernels are switched off");
  m.def("pack8", &pack8, "8 bit form of a tensor's rows");
  m.def("unpack8", &unpack8, "values of an 8 bit form");
  m.def("gelu8_forward", &gelu8_forward, "GELU, input kept in 8 bits");
  m.def("gelu8_backward", &gelu8_backward, "GELU from an 8 bit input");
  m.def("norm_forward", &norm_forward, "layer norm of rows");
  m.def("norm_backward", &norm_backward, "layer norm's gradients");
  m.def("weight_grad8", &weight_grad8, "dW, db from an 8 bit input");
}
