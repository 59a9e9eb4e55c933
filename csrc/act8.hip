// Activations in 8 bits: packing, unpacking, and GELU with its input kept
// that way (the form itself is described in act8.h).
//
// All four kernels are single passes bound by memory: a lane takes 8
// consecutive values of a row, so that a block of 64 is 8 neighbouring
// lanes and its maximum costs three register permutations.
//
// Measured in bf16, calls of one kind in a row: 16384 x 2304 packed in 19 us
// (5.9 TB/s, some of it from the last cache) and unpacked in 18 us, GELU of
// 16384 x 4096 forward with both 8 bit forms in 75 us (5.4 TB/s), backward in
// 63 us (5.4 TB/s). GELU's arithmetic takes about as long as its memory does.

#include "act8.h"

namespace kfac {

namespace {

constexpr int kThreads = 256;
constexpr int kRows = 2;  // that a thread takes one after the other

// A block covers 256 / L rows of L chunks, kRows times; L is a power of two,
// so that finding a thread's place takes shifts only.
struct Place {
  long R;
  int D;
  int blocks;  // exponents a row
  int shift;   // log2 L
};

struct Chunk {
  long row;  // the first one
  int step;  // to the next one
  int chunk;
  int n;     // how many of the chunk's 8 values are in a row
};

__device__ __forceinline__ Chunk chunk_of(const Place& p) {
  const int rows = kThreads >> p.shift;
  const int lane = threadIdx.x & ((1 << p.shift) - 1);
  Chunk c;
  c.row = (long)blockIdx.y * rows * kRows + (threadIdx.x >> p.shift);
  c.step = rows;
  c.chunk = (blockIdx.x << p.shift) + lane;
  c.n = p.D - c.chunk * kChunk;
  return c;
}

// TAIL: rows may end inside a chunk.
template <bool TAIL, typename T>
__device__ __forceinline__ void get(const T* p, int n, float v[8]) {
  if (TAIL) {
    load_chunk(p, n, v);
  } else {
    load8(p, v);
  }
}
template <bool TAIL, typename T>
__device__ __forceinline__ void put(T* p, int n, const float v[8]) {
  if (TAIL) {
    store_chunk(p, n, v);
  } else {
    store8(p, v);
  }
}

// All lanes of a block of 64 values call this, or none.
template <bool TAIL>
__device__ __forceinline__ void pack(
    const float v[8],
    const Place& p,
    const Chunk& c,
    long row,
    int8_t* codes,
    uint8_t* exps) {
  const bool any = c.n > 0;
  pack_chunk<false>(
      v, any, 0, TAIL ? c.n : kChunk, codes + row * p.D + c.chunk * kChunk,
      exps + row * p.blocks + c.chunk / 8, c.chunk % 8 == 0);
}

template <typename T, bool TAIL>
__global__ __launch_bounds__(kThreads) void pack8_kernel(
    const T* __restrict__ x,
    int8_t* __restrict__ codes,
    uint8_t* __restrict__ exps,
    Place p) {
  const Chunk c = chunk_of(p);
  float v[kRows][8] = {};
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const long row = c.row + i * c.step;
    if (row < p.R && c.n > 0) {
      get<TAIL>(x + row * p.D + c.chunk * kChunk, c.n, v[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const long row = c.row + i * c.step;
    if (row < p.R) pack<TAIL>(v[i], p, c, row, codes, exps);
  }
}

// The codes and the exponent of a chunk.
template <bool TAIL>
__device__ __forceinline__ void get_packed(
    const Place& p,
    const Chunk& c,
    long row,
    const int8_t* codes,
    const uint8_t* exps,
    float v[8]) {
  const int8_t* at = codes + row * p.D + c.chunk * kChunk;
  const unsigned byte = exps[row * p.blocks + c.chunk / 8];
  if (TAIL) {
    unpack_chunk(at, byte, c.n, v);
  } else {
    unpack8(at, byte, v);
  }
}

template <typename T, bool TAIL>
__global__ __launch_bounds__(kThreads) void unpack8_kernel(
    const int8_t* __restrict__ codes,
    const uint8_t* __restrict__ exps,
    T* __restrict__ out,
    Place p) {
  const Chunk c = chunk_of(p);
  if (c.n <= 0) return;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const long row = c.row + i * c.step;
    if (row >= p.R) return;
    float v[8];
    get_packed<TAIL>(p, c, row, codes, exps, v);
    put<TAIL>(out + row * p.D + c.chunk * kChunk, c.n, v);
  }
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
// evaluated in fp32. The exponential's argument is rounded three times, 1.5
// x^2 half steps of fp32: the tail as a whole is off by 5.5e-7 of itself up to
// |x| = 2, 8.4e-7 up to 4, 2.7e-6 up to 8 and 5.3e-6 up to 10, where it is
// 8e-24. One exponential, one reciprocal and 14 other operations; with the
// library's erfc these kernels were bound by arithmetic (16384 x 4096 bf16:
// 147 us forward, 157 us backward).
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
  if (TANH) return x * gate_of(x);
  float e;
  const float q = lower_tail(x, e);
  return x * (x < 0.f ? q : 1.f - q);
}

template <bool TANH>
__device__ __forceinline__ float gelu_slope(float x) {
  if (TANH) {
    const float p = gate_of(x);
    // p (1 - p) is 0 beyond |x| = 30, where x^2 may overflow
    const float c = __builtin_amdgcn_fmed3f(x, -30.f, 30.f);
    const float slope = kGate * fmaf(3.f * kCubic * c, c, 1.f);
    return fmaf(c * p * (1.f - p), slope, p);
  }
  float e;
  const float q = lower_tail(x, e);
  return fmaf(x * e, kInvSqrt2Pi, x < 0.f ? q : 1.f - q);
}

template <typename T, bool TANH, bool TAIL>
__global__ __launch_bounds__(kThreads) void gelu8_fwd_kernel(
    const T* __restrict__ x,
    T* __restrict__ y,
    int8_t* __restrict__ in_codes,  // may be null
    uint8_t* __restrict__ in_exps,
    int8_t* __restrict__ out_codes,  // may be null
    uint8_t* __restrict__ out_exps,
    Place p) {
  const Chunk c = chunk_of(p);
  float v[kRows][8] = {};
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const long row = c.row + i * c.step;
    if (row < p.R && c.n > 0) {
      get<TAIL>(x + row * p.D + c.chunk * kChunk, c.n, v[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const long row = c.row + i * c.step;
    if (row >= p.R) return;
    if (in_codes != nullptr) pack<TAIL>(v[i], p, c, row, in_codes, in_exps);
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
      v[i][j] = round_to(gelu_of<TANH>(v[i][j]), y);
    }
    if (c.n > 0) put<TAIL>(y + row * p.D + c.chunk * kChunk, c.n, v[i]);
    if (out_codes != nullptr) {
      pack<TAIL>(v[i], p, c, row, out_codes, out_exps);
    }
  }
}

template <typename T, bool TANH, bool TAIL>
__global__ __launch_bounds__(kThreads) void gelu8_bwd_kernel(
    const T* __restrict__ dy,
    const int8_t* __restrict__ codes,
    const uint8_t* __restrict__ exps,
    T* __restrict__ dx,
    Place p) {
  const Chunk c = chunk_of(p);
  if (c.n <= 0) return;
  float g[kRows][8], v[kRows][8];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const long row = c.row + i * c.step;
    if (row < p.R) {
      get<TAIL>(dy + row * p.D + c.chunk * kChunk, c.n, g[i]);
      get_packed<TAIL>(p, c, row, codes, exps, v[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const long row = c.row + i * c.step;
    if (row >= p.R) return;
#pragma unroll
    for (int j = 0; j < kChunk; ++j) g[i][j] *= gelu_slope<TANH>(v[i][j]);
    put<TAIL>(dx + row * p.D + c.chunk * kChunk, c.n, g[i]);
  }
}

// Calls fn(grid, place, first row, TAIL) for slabs of rows that a grid's
// second dimension can hold.
template <typename Fn>
hipError_t by_slabs(long R, int D, Fn fn) {
  const int blocks = ceil_div(D, kBlock8), chunks = blocks * 8;
  // the widest power of two that leaves no more than 1/16 of the lanes idle
  int shift = 8;
  while (shift > 3 &&
         (long)(ceil_div(chunks, 1 << shift) << shift) * 15 >
             (long)chunks * 16) {
    --shift;
  }
  const int rows = (kThreads >> shift) * kRows;
  const long most = 65535L * rows;
  for (long r = 0; r < R; r += most) {
    const long here = R - r < most ? R - r : most;
    const dim3 grid(
        ceil_div(chunks, 1 << shift), (unsigned)((here + rows - 1) / rows));
    const Place p{here, D, blocks, shift};
    if (D % kChunk) {
      fn(grid, p, r, std::true_type());
    } else {
      fn(grid, p, r, std::false_type());
    }
    KFAC_HIP_CHECK(hipGetLastError());
  }
  return hipSuccess;
}

}  // namespace

template <typename T>
hipError_t pack8_t(
    hipStream_t s,
    const T* x,
    int8_t* codes,
    uint8_t* exps,
    long R,
    int D) {
  return by_slabs(R, D, [&](dim3 grid, const Place& p, long r, auto tail) {
    pack8_kernel<T, decltype(tail)::value><<<grid, kThreads, 0, s>>>(
        x + r * D, codes + r * D, exps + r * p.blocks, p);
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
  return by_slabs(R, D, [&](dim3 grid, const Place& p, long r, auto tail) {
    unpack8_kernel<T, decltype(tail)::value><<<grid, kThreads, 0, s>>>(
        codes + r * D, exps + r * p.blocks, out + r * D, p);
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
  return by_slabs(R, D, [&](dim3 grid, const Place& p, long r, auto tail) {
    constexpr bool TAIL = decltype(tail)::value;
    auto kernel = tanh ? gelu8_fwd_kernel<T, true, TAIL>
                       : gelu8_fwd_kernel<T, false, TAIL>;
    kernel<<<grid, kThreads, 0, s>>>(
        x + r * D, y + r * D, ic == nullptr ? nullptr : ic + r * D,
        ic == nullptr ? nullptr : ie + r * p.blocks,
        oc == nullptr ? nullptr : oc + r * D,
        oc == nullptr ? nullptr : oe + r * p.blocks, p);
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
  return by_slabs(R, D, [&](dim3 grid, const Place& p, long r, auto tail) {
    constexpr bool TAIL = decltype(tail)::value;
    auto kernel = tanh ? gelu8_bwd_kernel<T, true, TAIL>
                       : gelu8_bwd_kernel<T, false, TAIL>;
    kernel<<<grid, kThreads, 0, s>>>(
        dy + r * D, codes + r * D, exps + r * p.blocks, dx + r * D, p);
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
