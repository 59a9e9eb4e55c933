// Activations in 8 bits: packing, unpacking, and GELU with its input kept
// that way (the form itself is described in act8.h).
//
// All four kernels are single passes bound by memory: a lane takes 8
// consecutive values of a row, so that a block of 64 is 8 neighbouring
// lanes and its maximum costs three register permutations.

#include "act8.h"

namespace kfac {

namespace {

constexpr int kThreads = 256;

// Rows are padded to whole blocks of lanes: unit u is chunk u % upr of row
// u / upr, upr a multiple of 8.
struct Unit {
  long row;
  int chunk;
  int n;  // how many of the chunk's 8 values are in the row
};

__device__ __forceinline__ Unit unit_of(unsigned u, unsigned upr, int D) {
  const unsigned row = u / upr;
  const unsigned chunk = u - row * upr;
  return {(long)row, (int)chunk, D - (int)chunk * kChunk};
}

template <typename T>
__global__ __launch_bounds__(kThreads) void pack8_kernel(
    const T* __restrict__ x,
    int8_t* __restrict__ codes,
    uint8_t* __restrict__ exps,
    unsigned units,
    unsigned upr,
    int D,
    int blocks) {
  const unsigned u = blockIdx.x * kThreads + threadIdx.x;
  if (u >= units) return;  // whole blocks: upr is a multiple of 8
  const Unit t = unit_of(u, upr, D);
  const long at = t.row * D + t.chunk * kChunk;
  float v[8];
  load_chunk(x + at, t.n, v);
  pack_chunk(
      v, 0, t.n, codes + at, exps + t.row * blocks + t.chunk / 8,
      t.chunk % 8 == 0);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void unpack8_kernel(
    const int8_t* __restrict__ codes,
    const uint8_t* __restrict__ exps,
    T* __restrict__ out,
    unsigned units,
    unsigned upr,
    int D,
    int blocks) {
  const unsigned u = blockIdx.x * kThreads + threadIdx.x;
  if (u >= units) return;
  const Unit t = unit_of(u, upr, D);
  if (t.n <= 0) return;
  const long at = t.row * D + t.chunk * kChunk;
  float v[8];
  unpack_chunk(codes + at, exps[t.row * blocks + t.chunk / 8], t.n, v);
  store_chunk(out + at, t.n, v);
}

// GELU: y = x * P(x) with P the normal distribution function, or its tanh
// form, a logistic gate: (1 + tanh u) / 2 = 1 / (1 + exp(-2u)).
constexpr float kInvSqrt2Pi = 0.3989422804014327f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kGate = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kCubic = 0.044715f;

// P(-|x|) = exp(-x^2 / 2) * m(|x|), and the exponential. m, Mills' ratio
// over sqrt(2 pi), is smooth and falls like 1 / |x|: a polynomial of degree
// 7 in 1 / (1 + 0.34 |x|), fitted by reweighted least squares for an even
// relative error up to |x| = 10, is off by 1.4e-7, and by 5e-7 when it is
// evaluated in fp32. One exponential, one reciprocal and 14 other
// operations; with the library's erfc these kernels were bound by
// arithmetic (16384 x 4096 bf16: 147 us forward, 157 us backward).
__device__ __forceinline__ float lower_tail(float x, float& exponential) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.34f, fabsf(x), 1.f));
  float m = 0.0489479969f;
  m = fmaf(m, t, -0.218984677f);
  m = fmaf(m, t, 0.298419536f);
  m = fmaf(m, t, -0.0649849661f);
  m = fmaf(m, t, 0.176260347f);
  m = fmaf(m, t, 0.123280336f);
  m = fmaf(m, t, 0.137138441f);
  m = fmaf(m, t, -7.70223557e-05f);
  exponential = __builtin_amdgcn_exp2f(x * x * (-0.5f * kLog2e));
  return exponential * m;
}

__device__ __forceinline__ float gate_of(float x) {
  const float u = x * fmaf(kGate * kCubic * kLog2e, x * x, kGate * kLog2e);
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-u));
}

template <bool TANH>
__device__ __forceinline__ float gelu_of(float x) {
  // below -100 the gate is 0: so is the result, at minus infinity too
  if (TANH) return fmaxf(x, -100.f) * gate_of(x);
  float e;
  const float q = lower_tail(x, e);
  return fmaf(-fminf(fabsf(x), 100.f), q, fmaxf(x, 0.f));
}

template <bool TANH>
__device__ __forceinline__ float gelu_slope(float x) {
  if (TANH) {
    const float p = gate_of(x);
    // p (1 - p) is 0 beyond |x| = 30, where x^2 may overflow
    const float c = fminf(fmaxf(x, -30.f), 30.f);
    const float slope = kGate * fmaf(3.f * kCubic * c, c, 1.f);
    return fmaf(c * p * (1.f - p), slope, p);
  }
  float e;
  const float q = lower_tail(x, e);
  return fmaf(x * e, kInvSqrt2Pi, x < 0.f ? q : 1.f - q);
}

template <typename T, bool TANH>
__global__ __launch_bounds__(kThreads) void gelu8_fwd_kernel(
    const T* __restrict__ x,
    T* __restrict__ y,
    int8_t* __restrict__ in_codes,  // may be null
    uint8_t* __restrict__ in_exps,
    int8_t* __restrict__ out_codes,  // may be null
    uint8_t* __restrict__ out_exps,
    unsigned units,
    unsigned upr,
    int D,
    int blocks) {
  const unsigned u = blockIdx.x * kThreads + threadIdx.x;
  if (u >= units) return;
  const Unit t = unit_of(u, upr, D);
  const long at = t.row * D + t.chunk * kChunk;
  const long block = t.row * blocks + t.chunk / 8;
  const bool first = t.chunk % 8 == 0;
  float v[8];
  load_chunk(x + at, t.n, v);
  if (in_codes != nullptr) {
    pack_chunk(v, 0, t.n, in_codes + at, in_exps + block, first);
  }
#pragma unroll
  for (int j = 0; j < kChunk; ++j) v[j] = round_to(gelu_of<TANH>(v[j]), y);
  store_chunk(y + at, t.n, v);
  if (out_codes != nullptr) {
    pack_chunk(v, 0, t.n, out_codes + at, out_exps + block, first);
  }
}

template <typename T, bool TANH>
__global__ __launch_bounds__(kThreads) void gelu8_bwd_kernel(
    const T* __restrict__ dy,
    const int8_t* __restrict__ codes,
    const uint8_t* __restrict__ exps,
    T* __restrict__ dx,
    unsigned units,
    unsigned upr,
    int D,
    int blocks) {
  const unsigned u = blockIdx.x * kThreads + threadIdx.x;
  if (u >= units) return;
  const Unit t = unit_of(u, upr, D);
  if (t.n <= 0) return;
  const long at = t.row * D + t.chunk * kChunk;
  float g[8], v[8];
  load_chunk(dy + at, t.n, g);
  unpack_chunk(codes + at, exps[t.row * blocks + t.chunk / 8], t.n, v);
#pragma unroll
  for (int j = 0; j < kChunk; ++j) g[j] *= gelu_slope<TANH>(v[j]);
  store_chunk(dx + at, t.n, g);
}

// Calls fn(first row, rows, units, upr) for slabs of rows whose units fit
// 31 bits (a tensor of more than 2^34 values takes several launches).
template <typename Fn>
hipError_t by_slabs(long R, int D, Fn fn) {
  const long upr = (long)ceil_div(D, kBlock8) * 8;
  const long most = (1L << 31) / upr - 1;
  for (long r = 0; r < R; r += most) {
    const long rows = R - r < most ? R - r : most;
    fn(r, (unsigned)(rows * upr), (unsigned)upr);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

unsigned grid_of(unsigned units) { return (units + kThreads - 1) / kThreads; }

}  // namespace

template <typename T>
hipError_t pack8_t(
    hipStream_t s,
    const T* x,
    int8_t* codes,
    uint8_t* exps,
    long R,
    int D) {
  const int blocks = ceil_div(D, kBlock8);
  return by_slabs(R, D, [&](long r, unsigned units, unsigned upr) {
    pack8_kernel<T><<<grid_of(units), kThreads, 0, s>>>(
        x + r * D, codes + r * D, exps + r * blocks, units, upr, D, blocks);
  });
}

template <typename T>
hipError_t unpack8_t(
    hipStream_t s,
    const int8_t* codes,
    const uint8_t* exps,
    T* out,
    long R,
    int D) {
  const int blocks = ceil_div(D, kBlock8);
  return by_slabs(R, D, [&](long r, unsigned units, unsigned upr) {
    unpack8_kernel<T><<<grid_of(units), kThreads, 0, s>>>(
        codes + r * D, exps + r * blocks, out + r * D, units, upr, D, blocks);
  });
}

template <typename T>
hipError_t gelu8_fwd_t(
    hipStream_t s,
    const T* x,
    T* y,
    int8_t* ic,
    uint8_t* ie,
    int8_t* oc,
    uint8_t* oe,
    long R,
    int D,
    bool tanh) {
  const int blocks = ceil_div(D, kBlock8);
  auto kernel = tanh ? gelu8_fwd_kernel<T, true> : gelu8_fwd_kernel<T, false>;
  return by_slabs(R, D, [&](long r, unsigned units, unsigned upr) {
    kernel<<<grid_of(units), kThreads, 0, s>>>(
        x + r * D, y + r * D, ic == nullptr ? nullptr : ic + r * D,
        ic == nullptr ? nullptr : ie + r * blocks,
        oc == nullptr ? nullptr : oc + r * D,
        oc == nullptr ? nullptr : oe + r * blocks, units, upr, D, blocks);
  });
}

template <typename T>
hipError_t gelu8_bwd_t(
    hipStream_t s,
    const T* dy,
    const int8_t* codes,
    const uint8_t* exps,
    T* dx,
    long R,
    int D,
    bool tanh) {
  const int blocks = ceil_div(D, kBlock8);
  auto kernel = tanh ? gelu8_bwd_kernel<T, true> : gelu8_bwd_kernel<T, false>;
  return by_slabs(R, D, [&](long r, unsigned units, unsigned upr) {
    kernel<<<grid_of(units), kThreads, 0, s>>>(
        dy + r * D, codes + r * D, exps + r * blocks, dx + r * D, units, upr,
        D, blocks);
  });
}

#define KFAC_ACT8(T)                                                          \
  template hipError_t pack8_t<T>(                                             \
      hipStream_t, const T*, int8_t*, uint8_t*, long, int);                   \
  template hipError_t unpack8_t<T>(                                           \
      hipStream_t, const int8_t*, const uint8_t*, T*, long, int);             \
  template hipError_t gelu8_fwd_t<T>(                                         \
      hipStream_t, const T*, T*, int8_t*, uint8_t*, int8_t*, uint8_t*, long,  \
      int, bool);                                                             \
  template hipError_t gelu8_bwd_t<T>(                                         \
      hipStream_t, const T*, const int8_t*, const uint8_t*, T*, long, int,    \
      bool);
KFAC_ACT8(float)
KFAC_ACT8(__hip_bfloat16)
KFAC_ACT8(__half)
#undef KFAC_ACT8

}  // namespace kfac
