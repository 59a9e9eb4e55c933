// Python binding of the transformer block's training kernels.
//
// Host-side glue only: checks that keep the kernels inside their tensors,
// allocation, launches on the current stream of the tensors' device. All
// tensors are contiguous here; the callers in kfac_amd.ops see to that.

#include "training.h"

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <tuple>

namespace {

using torch::Tensor;
using OptTensor = std::optional<Tensor>;

#define CHECK_OK(expr)                                                       \
  do {                                                                       \
    hipError_t _e = (expr);                                                  \
    TORCH_CHECK(_e == hipSuccess, "HIP error: ", hipGetErrorString(_e));     \
  } while (0)

hipStream_t stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

void check(const Tensor& t, const char* name, const Tensor& like) {
  TORCH_CHECK(t.is_cuda(), name, " must be a GPU tensor");
  TORCH_CHECK(t.device() == like.device(), name, " is on another device");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

int type_of(torch::ScalarType st) {
  switch (st) {
    case torch::kFloat32:
      return kfac::kF32;
    case torch::kBFloat16:
      return kfac::kBF16;
    case torch::kFloat16:
      return kfac::kF16;
    default:
      TORCH_CHECK(false, "unsupported dtype: ", st);
  }
}

// Calls fn with a value of the C++ type.
template <typename Fn>
void by_type(torch::ScalarType st, Fn fn) {
  switch (type_of(st)) {
    case kfac::kF32:
      return fn(float());
    case kfac::kBF16:
      return fn(__hip_bfloat16());
    default:
      return fn(__half());
  }
}

struct Shape {
  long R;
  int D;
  long blocks;
};

Shape rows_of(const Tensor& t) {
  TORCH_CHECK(t.dim() >= 1, "a tensor of rows has a dimension or more");
  const long D = t.size(-1);
  TORCH_CHECK(D > 0 && D < (1L << 30), "rows of 1 to 2^30 - 1 values");
  return {t.numel() / D, (int)D, (D + kfac::kBlock8 - 1) / kfac::kBlock8};
}

// The two tensors of the 8 bit form of `like`.
std::tuple<Tensor, Tensor> empty_packed(const Tensor& like, long blocks) {
  auto size = like.sizes().vec();
  auto codes = torch::empty(size, like.options().dtype(torch::kInt8));
  size.back() = blocks;
  return {codes, torch::empty(size, like.options().dtype(torch::kUInt8))};
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
      out.push_back(c);
      out.push_back(e);
    }
  }
};

Shape check_packed(
    const Tensor& codes,
    const Tensor& exps,
    const Tensor& like) {
  check(codes, "codes", like);
  check(exps, "exponents", like);
  TORCH_CHECK(codes.scalar_type() == torch::kInt8, "codes must be int8");
  TORCH_CHECK(exps.scalar_type() == torch::kUInt8, "exponents must be uint8");
  const Shape s = rows_of(codes);
  TORCH_CHECK(
      exps.numel() == s.R * s.blocks, "codes and exponents do not match");
  return s;
}

std::tuple<Tensor, Tensor> pack8(Tensor x) {
  check(x, "x", x);
  const c10::DeviceGuard guard(x.device());
  const Shape s = rows_of(x);
  auto [codes, exps] = empty_packed(x, s.blocks);
  if (s.R > 0) {
    by_type(x.scalar_type(), [&](auto t) {
      using T = decltype(t);
      CHECK_OK(kfac::pack8_t<T>(
          stream_of(x), (const T*)x.const_data_ptr(),
          (int8_t*)codes.data_ptr(), (uint8_t*)exps.data_ptr(), s.R, s.D));
    });
  }
  return {codes, exps};
}

Tensor unpack8(Tensor codes, Tensor exps, torch::ScalarType dtype) {
  const Shape s = check_packed(codes, exps, codes);
  const c10::DeviceGuard guard(codes.device());
  auto out = torch::empty(codes.sizes(), codes.options().dtype(dtype));
  if (s.R > 0) {
    by_type(dtype, [&](auto t) {
      using T = decltype(t);
      CHECK_OK(kfac::unpack8_t<T>(
          stream_of(codes), (const int8_t*)codes.const_data_ptr(),
          (const uint8_t*)exps.const_data_ptr(), (T*)out.data_ptr(), s.R,
          s.D));
    });
  }
  return out;
}

// (y[, codes and exponents of x][, of y])
std::vector<Tensor> gelu8_forward(
    Tensor x,
    bool tanh,
    bool pack_input,
    bool pack_output) {
  check(x, "x", x);
  const c10::DeviceGuard guard(x.device());
  const Shape s = rows_of(x);
  auto y = torch::empty_like(x);
  std::vector<Tensor> out{y};
  const Packs packs(x, s.blocks, pack_input, pack_output, out);
  if (s.R > 0) {
    by_type(x.scalar_type(), [&](auto t) {
      using T = decltype(t);
      CHECK_OK(kfac::gelu8_fwd_t<T>(
          stream_of(x), (const T*)x.const_data_ptr(), (T*)y.data_ptr(),
          packs.codes[0], packs.exps[0], packs.codes[1], packs.exps[1], s.R,
          s.D, tanh));
    });
  }
  return out;
}

Tensor gelu8_backward(Tensor dy, Tensor codes, Tensor exps, bool tanh) {
  check(dy, "dy", dy);
  const Shape s = check_packed(codes, exps, dy);
  TORCH_CHECK(dy.sizes() == codes.sizes(), "dy and the input do not match");
  const c10::DeviceGuard guard(dy.device());
  auto dx = torch::empty_like(dy);
  if (s.R > 0) {
    by_type(dy.scalar_type(), [&](auto t) {
      using T = decltype(t);
      CHECK_OK(kfac::gelu8_bwd_t<T>(
          stream_of(dy), (const T*)dy.const_data_ptr(),
          (const int8_t*)codes.const_data_ptr(),
          (const uint8_t*)exps.const_data_ptr(), (T*)dx.data_ptr(), s.R, s.D,
          tanh));
    });
  }
  return dx;
}

// Calls fn with values of both types: the same, or one of them fp32.
template <typename Fn>
void by_types(torch::ScalarType x, torch::ScalarType y, Fn fn) {
  by_type(x, [&](auto tx) {
    using TX = decltype(tx);
    if (x == y) {
      fn(tx, tx);
    } else if (y == torch::kFloat32) {
      fn(tx, float());
    } else if constexpr (std::is_same_v<TX, float>) {
      by_type(y, [&](auto ty) { fn(tx, ty); });
    } else {
      TORCH_CHECK(false, "no layer norm between ", x, " and ", y);
    }
  });
}

const void* ptr_or_null(const OptTensor& t) {
  return t ? t->const_data_ptr() : nullptr;
}
int type_or_f32(const OptTensor& t) {
  return t ? type_of(t->scalar_type()) : kfac::kF32;
}

void check_param(const OptTensor& t, const char* name, const Tensor& x) {
  if (!t) return;
  check(*t, name, x);
  TORCH_CHECK(t->numel() == x.size(-1), name, " does not fit the rows");
}

// (y, total or x, mean, rstd[, codes, exponents of the input][, of the
// output])
std::vector<Tensor> norm_forward(
    Tensor x,
    OptTensor r,
    OptTensor w,
    OptTensor b,
    double eps,
    torch::ScalarType dtype,
    bool pack_input,
    bool pack_output) {
  check(x, "x", x);
  const c10::DeviceGuard guard(x.device());
  const Shape s = rows_of(x);
  check_param(w, "weight", x);
  check_param(b, "bias", x);
  if (r) {
    check(*r, "residual", x);
    TORCH_CHECK(r->sizes() == x.sizes(), "x and residual do not match");
  }
  auto y = torch::empty(x.sizes(), x.options().dtype(dtype));
  auto total = r ? torch::empty_like(x) : x;
  auto mean = torch::empty({s.R}, x.options().dtype(torch::kFloat32));
  auto rstd = torch::empty_like(mean);
  std::vector<Tensor> out{y, total, mean, rstd};
  const Packs packs(x, s.blocks, pack_input, pack_output, out);
  if (s.R > 0) {
    by_types(x.scalar_type(), dtype, [&](auto tx, auto ty) {
      using TX = decltype(tx);
      using TY = decltype(ty);
      CHECK_OK((kfac::norm_fwd_t<TX, TY>(
          stream_of(x), (const TX*)x.const_data_ptr(), ptr_or_null(r),
          type_or_f32(r), ptr_or_null(w), type_or_f32(w), ptr_or_null(b),
          type_or_f32(b), r ? (TX*)total.data_ptr() : nullptr,
          (TY*)y.data_ptr(), mean.data_ptr<float>(), rstd.data_ptr<float>(),
          packs.codes[0], packs.exps[0], packs.codes[1], packs.exps[1], s.R,
          s.D, (float)eps)));
    });
  }
  return out;
}

// (dx, dweight or None, dbias or None); x or (codes, exps)
std::tuple<Tensor, OptTensor, OptTensor> norm_backward(
    Tensor dy,
    OptTensor x,
    OptTensor codes,
    OptTensor exps,
    Tensor mean,
    Tensor rstd,
    OptTensor w,
    bool want_dw,
    bool want_db,
    OptTensor dt,
    torch::ScalarType dtype) {
  check(dy, "dy", dy);
  const c10::DeviceGuard guard(dy.device());
  const Shape s = rows_of(dy);
  if (x) {
    check(*x, "x", dy);
    TORCH_CHECK(
        x->sizes() == dy.sizes() && x->scalar_type() == dtype,
        "x and dy do not match");
  } else {
    TORCH_CHECK(codes && exps, "x or its 8 bit form");
    check_packed(*codes, *exps, dy);
    TORCH_CHECK(codes->sizes() == dy.sizes(), "x and dy do not match");
  }
  check(mean, "mean", dy);
  check(rstd, "rstd", dy);
  TORCH_CHECK(
      mean.scalar_type() == torch::kFloat32 &&
          rstd.scalar_type() == torch::kFloat32 && mean.numel() == s.R &&
          rstd.numel() == s.R,
      "mean and rstd must be fp32, one a row");
  check_param(w, "weight", dy);
  if (dt) {
    check(*dt, "grad_total", dy);
    TORCH_CHECK(
        dt->sizes() == dy.sizes() && dt->scalar_type() == dtype,
        "grad_total and dx do not match");
  }
  auto dx = torch::empty(dy.sizes(), dy.options().dtype(dtype));
  const auto ptype = w ? w->scalar_type() : torch::kFloat32;
  const auto popts = dy.options().dtype(ptype);
  OptTensor dw, db;
  const std::vector<int64_t> size{s.D};
  if (want_dw) dw = s.R ? torch::empty(size, popts) : torch::zeros(size, popts);
  if (want_db) db = s.R ? torch::empty(size, popts) : torch::zeros(size, popts);
  if (s.R == 0) return {dx, dw, db};
  Tensor partial;
  if (want_dw || want_db) {
    partial = torch::empty(
        {(long)kfac::norm_bwd_partials(s.R, s.D) * 2 * s.D},
        dy.options().dtype(torch::kFloat32));
  }
  by_types(dtype, dy.scalar_type(), [&](auto tx, auto ty) {
    using TX = decltype(tx);
    using TY = decltype(ty);
    CHECK_OK((kfac::norm_bwd_t<TX, TY>(
        stream_of(dy), (const TY*)dy.const_data_ptr(),
        (const TX*)ptr_or_null(x), (const int8_t*)ptr_or_null(codes),
        (const uint8_t*)ptr_or_null(exps), mean.data_ptr<float>(),
        rstd.data_ptr<float>(), ptr_or_null(w), type_or_f32(w),
        (const TX*)ptr_or_null(dt), (TX*)dx.data_ptr(),
        partial.defined() ? partial.data_ptr<float>() : nullptr,
        dw ? dw->data_ptr() : nullptr, type_of(ptype),
        db ? db->data_ptr() : nullptr, type_of(ptype), s.R, s.D)));
  });
  return {dx, dw, db};
}

// (dW, db or None)
std::tuple<Tensor, OptTensor> weight_grad8(
    Tensor g,
    Tensor codes,
    Tensor exps,
    bool want_bias,
    torch::ScalarType dtype) {
  check(g, "g", g);
  const c10::DeviceGuard guard(g.device());
  const Shape sx = check_packed(codes, exps, g);
  const Shape sg = rows_of(g);
  TORCH_CHECK(sx.R == sg.R, "the gradient and the input have other rows");
  const long M = sg.R;
  const long N = sg.D, K = sx.D;
  const auto opts = g.options().dtype(dtype);
  const auto f32 = g.options().dtype(torch::kFloat32);
  const std::vector<int64_t> size{N, K}, bias_size{N};
  OptTensor db;
  if (M == 0) {
    if (want_bias) db = torch::zeros(bias_size, opts);
    return {torch::zeros(size, opts), db};
  }
  kfac::WGradPlan plan;
  by_type(g.scalar_type(), [&](auto t) {
    plan = kfac::wgrad8_plan<decltype(t)>(M, sg.D, sx.D);
  });
  const long rows = (long)plan.splits * plan.tiles_k;
  auto dw = torch::empty(size, opts);
  if (want_bias) db = torch::empty(bias_size, opts);
  // a single fp32 sum is the result itself
  const bool direct = plan.splits == 1 && dtype == torch::kFloat32;
  const bool bias_direct = rows == 1 && dtype == torch::kFloat32;
  Tensor sums = dw, bias = want_bias ? *db : Tensor();
  if (!direct) {
    sums = torch::empty({plan.splits * N * K}, f32);
  }
  if (want_bias && !bias_direct) bias = torch::empty({rows * N}, f32);
  const auto stream = stream_of(g);
  by_type(g.scalar_type(), [&](auto t) {
    using T = decltype(t);
    CHECK_OK(kfac::wgrad8_t<T>(
        stream, (const T*)g.const_data_ptr(),
        (const int8_t*)codes.const_data_ptr(),
        (const uint8_t*)exps.const_data_ptr(), M, sg.D, sx.D, plan,
        sums.data_ptr<float>(),
        want_bias ? bias.data_ptr<float>() : nullptr));
  });
  const bool add_bias = want_bias && !bias_direct;
  CHECK_OK(kfac::wgrad8_add(
      stream, sums.data_ptr<float>(), plan.splits, N * K,
      direct ? nullptr : dw.data_ptr(),
      add_bias ? bias.data_ptr<float>() : nullptr, (int)rows, N,
      add_bias ? db->data_ptr() : nullptr, type_of(dtype)));
  return {dw, db};
}

}  // namespace

void bind_training(pybind11::module& m) {
  m.def("pack8", &pack8, "8 bit form of a tensor's rows");
  m.def("unpack8", &unpack8, "values of an 8 bit form");
  m.def("gelu8_forward", &gelu8_forward, "GELU, input kept in 8 bits");
  m.def("gelu8_backward", &gelu8_backward, "GELU from an 8 bit input");
  m.def("norm_forward", &norm_forward, "layer norm of rows");
  m.def("norm_backward", &norm_backward, "layer norm's gradients");
  m.def("weight_grad8", &weight_grad8, "dW, db from an 8 bit input");
}
