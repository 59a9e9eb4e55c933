// Weight and bias gradient of a linear layer whose input was kept in 8 bits:
//
//   dW[n][k] = sum over tokens m of g[m][n] * a[m][k],  a = code * 2^e
//   db[n]    = sum over tokens m of g[m][n]
//
// A product over the tokens, the slow axis of both operands. A code times
// its power of two is exact in bf16, and so is a bf16 gradient; an fp16
// gradient is the sum of two bf16 numbers and an fp32 one of three (hi +
// mid + lo, 24 bits), so every product that the matrix cores see is exact
// and only the fp32 accumulation rounds, for each type of gradient.
//
// Tiles go from memory through registers, where codes become bf16 and
// gradients are split, into LDS as [token][column] images, two of them in
// turn, with one barrier a stage. ds_read_b64_tr_b16 hands a lane four
// tokens of one column, which is the fragment that mfma_f32_32x32x16_bf16
// wants, so nothing is transposed by hand.
//
// The tokens are split over blocks when the output has too few tiles to
// fill the card; the splits' fp32 sums are added by a second kernel in a
// fixed order.

#include <type_traits>

#include "act8.h"

namespace kfac {

namespace {

typedef __attribute__((ext_vector_type(4))) short short4v;
typedef __attribute__((ext_vector_type(16))) float f32x16;

struct WGrad {
  const void* g;         // [M][N]
  const int8_t* codes;   // [M][K]
  const uint8_t* exps;   // [M][blocks]
  float* out;            // [S][N][K]
  float* bias;           // [S * tiles_k][N], may be null
  long M;
  int N, K, blocks;
  int tiles_n, tiles_k;
  long rows;  // tokens of a split, a multiple of the stage
};

// 16 byte chunk c of row r: the 64 byte group is swapped by the row, so
// that the four rows of a transposed read lie in different banks.
template <int WIDTH>
__device__ __forceinline__ int slot(int r, int c) {
  return r * (WIDTH / 8) + (c ^ ((r & 3) << 2));
}

// Lane's 8 tokens (8 * (lane / 32) + j) of column col + lane % 32.
template <int WIDTH>
__device__ __forceinline__ bf16x8 fragment(
    const short* lds,
    int row,
    int col,
    int lane) {
  const int i = lane % 16;
  const int r = row + lane / 32 * 8 + i / 4;
  const int c = col + lane / 16 % 2 * 16 + i % 4 * 4;
  typedef __attribute__((address_space(3))) short4v* Ptr;
  const int half = c % 8;
  const short4v a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (Ptr)(lds + slot<WIDTH>(r, c / 8) * 8 + half));
  const short4v b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (Ptr)(lds + slot<WIDTH>(r + 4, c / 8) * 8 + half));
  typedef __attribute__((ext_vector_type(8))) short short8v;
  const short8v v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_bit_cast(bf16x8, v);
}

__device__ __forceinline__ unsigned high_halves(float lo, float hi) {
  // bytes 2, 3 of both: exact, since the values have 8 bits or fewer
  return __builtin_amdgcn_perm(
      __float_as_uint(hi), __float_as_uint(lo), 0x07060302);
}

// 8 gradients as they are in memory, the missing ones 0.
template <typename TG>
struct Raw {
  unsigned v[2 * sizeof(TG)];

  __device__ __forceinline__ void load(const TG* p, int n) {
    if (n >= kChunk) {
      __builtin_memcpy(v, p, sizeof(v));
    } else {
      TG t[8];
#pragma unroll
      for (int j = 0; j < kChunk; ++j) t[j] = j < n ? p[j] : (TG)0.f;
      __builtin_memcpy(v, t, sizeof(v));
    }
  }
  __device__ __forceinline__ void values(float f[8]) const {
    TG t[8];
    __builtin_memcpy(t, v, sizeof(v));
#pragma unroll
    for (int j = 0; j < kChunk; ++j) f[j] = load1(t + j);
  }
};

// Takes the leading 8 bits of each of 8 values off as bf16. Cut, not
// rounded: the rest is exact, and nothing overflows. An infinity leaves
// nothing, a NaN a NaN.
__device__ __forceinline__ void take_part(float v[8], unsigned part[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) part[j] = high_halves(v[2 * j], v[2 * j + 1]);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float top = __uint_as_float(__float_as_uint(v[j]) & 0xFFFF0000);
    v[j] = fabsf(v[j]) == __builtin_inff() ? 0.f : v[j] - top;
  }
}

template <typename TG, int NP, int BN, int BK, int BM, int WN, int WK>
__global__ __launch_bounds__(WN * WK * kWave) void wgrad8_kernel(WGrad a) {
  constexpr int kT = WN * WK * kWave;
  constexpr int TN = BN / WN, TK = BK / WK;        // a wave's part
  constexpr int FN = TN / 32, FK = TK / 32;        // in fragments
  constexpr int GC = BM * BN / 8 / kT;             // chunks a thread, g
  constexpr int XC = BM * BK / 16 / kT;            // 16 codes each
  constexpr int kImage = BM * (NP * BN + BK);      // of one stage
  static_assert(GC * kT * 8 == BM * BN && XC * kT * 16 == BM * BK, "");
  static_assert(kT % (BN / 8) == 0, "a thread keeps its columns");
  __shared__ __attribute__((aligned(16))) short lds[2 * kImage];

  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int tiles = a.tiles_n * a.tiles_k;
  const int split = blockIdx.x / tiles, tile = blockIdx.x % tiles;
  const int tk = tile % a.tiles_k, tn = tile / a.tiles_k;
  const int n0 = tn * BN, k0 = tk * BK;
  const long m0 = split * a.rows;
  const long m1 = m0 + a.rows < a.M ? m0 + a.rows : a.M;
  const int stages = (int)((m1 - m0 + BM - 1) / BM);
  const TG* g = (const TG*)a.g;

  f32x16 acc[FN][FK];
#pragma unroll
  for (int i = 0; i < FN; ++i) {
#pragma unroll
    for (int j = 0; j < FK; ++j) acc[i][j] = (f32x16)(0.f);
  }
  float bias[8] = {};

  Raw<TG> gv[GC];
  unsigned char xv[XC][16];
  unsigned xe[XC];
  const auto load = [&](int stage) {
    const long m = m0 + (long)stage * BM;
#pragma unroll
    for (int i = 0; i < GC; ++i) {
      const int c = tid + i * kT;
      const long row = m + c / (BN / 8);
      const int col = n0 + c % (BN / 8) * 8;
      gv[i].load(g + row * a.N + col, row < m1 ? a.N - col : 0);
    }
#pragma unroll
    for (int i = 0; i < XC; ++i) {
      const int c = tid + i * kT;
      const long row = m + c / (BK / 16);
      const int col = k0 + c % (BK / 16) * 16;
      const int n = row < m1 ? a.K - col : 0;
      const int8_t* p = a.codes + row * a.K + col;
      xe[i] = n > 0 ? a.exps[row * a.blocks + col / kBlock8] : 1;
      if (n >= 16) {
        __builtin_memcpy(xv[i], p, 16);
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) xv[i][j] = j < n ? p[j] : 0;
      }
    }
  };
  const auto put = [&](int stage) {
    short* gl = lds + (stage & 1) * kImage;
    short* xl = gl + NP * BM * BN;
    const bool sum = a.bias != nullptr && stage % a.tiles_k == tk;
#pragma unroll
    for (int i = 0; i < GC; ++i) {
      const int c = tid + i * kT;
      const int at = slot<BN>(c / (BN / 8), c % (BN / 8)) * 8;
      if (NP == 1) __builtin_memcpy(gl + at, gv[i].v, 16);
      if (NP == 1 && !sum) continue;
      float v[8];
      gv[i].values(v);
      if (sum) {
#pragma unroll
        for (int j = 0; j < 8; ++j) bias[j] += v[j];
      }
      if (NP == 1) continue;
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        unsigned part[4];
        take_part(v, part);
        __builtin_memcpy(gl + p * BM * BN + at, part, 16);
      }
    }
#pragma unroll
    for (int i = 0; i < XC; ++i) {
      const int c = tid + i * kT;
      const int row = c / (BK / 16), chunk = c % (BK / 16) * 2;
      const float s = scale_of(xe[i]);
      unsigned v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = high_halves(
            (float)(int8_t)xv[i][2 * j] * s,
            (float)(int8_t)xv[i][2 * j + 1] * s);
      }
      __builtin_memcpy(xl + slot<BK>(row, chunk) * 8, v, 16);
      __builtin_memcpy(xl + slot<BK>(row, chunk + 1) * 8, v + 4, 16);
    }
  };

  const int wn = wave / WK * TN, wk = wave % WK * TK;
  if (stages > 0) {
    load(0);
    put(0);
  }
  for (int stage = 0; stage < stages; ++stage) {
    if (stage + 1 < stages) load(stage + 1);
    __syncthreads();
    const short* gl = lds + (stage & 1) * kImage;
    const short* xl = gl + NP * BM * BN;
#pragma unroll
    for (int r = 0; r < BM; r += 16) {
      bf16x8 x[FK];
#pragma unroll
      for (int j = 0; j < FK; ++j) {
        x[j] = fragment<BK>(xl, r, wk + j * 32, lane);
      }
#pragma unroll
      for (int p = 0; p < NP; ++p) {
#pragma unroll
        for (int i = 0; i < FN; ++i) {
          const bf16x8 f =
              fragment<BN>(gl + p * BM * BN, r, wn + i * 32, lane);
#pragma unroll
          for (int j = 0; j < FK; ++j) {
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                f, x[j], acc[i][j], 0, 0, 0);
          }
        }
      }
    }
    if (stage + 1 < stages) put(stage + 1);
  }

  // column lane % 32, rows 8 * (r / 4) + 4 * (lane / 32) + r % 4
  float* out = a.out + (long)split * a.N * a.K;
#pragma unroll
  for (int i = 0; i < FN; ++i) {
#pragma unroll
    for (int j = 0; j < FK; ++j) {
      const int k = k0 + wk + j * 32 + lane % 32;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int n = n0 + wn + i * 32 + r / 4 * 8 + lane / 32 * 4 + r % 4;
        if (n < a.N && k < a.K) out[(long)n * a.K + k] = acc[i][j][r];
      }
    }
  }
  if (a.bias != nullptr) {
    // the threads that share columns, added in their order
    float* sums = (float*)lds;
    __syncthreads();
    const int chunk = tid % (BN / 8), part = tid / (BN / 8);
#pragma unroll
    for (int j = 0; j < 8; ++j) sums[part * BN + chunk * 8 + j] = bias[j];
    __syncthreads();
    for (int c = tid; c < BN; c += kT) {
      float s = 0.f;
      for (int i = 0; i < kT / (BN / 8); ++i) s += sums[i * BN + c];
      if (n0 + c < a.N) {
        a.bias[((long)split * a.tiles_k + tk) * a.N + n0 + c] = s;
      }
    }
  }
}

// out[i] = sum over S of parts[s][i], 4 values a thread
__global__ __launch_bounds__(256) void wgrad8_add_kernel(
    const float* __restrict__ parts,
    int S,
    long n,
    void* out,
    int type) {
  const long at = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= n) return;
  const int live = n - at < 4 ? (int)(n - at) : 4;
  float s[4] = {};
  if (live == 4) {
#pragma unroll 4
    for (int p = 0; p < S; ++p) {
      float v[4];
      __builtin_memcpy(v, parts + p * n + at, 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] += v[j];
    }
  } else {
    for (int p = 0; p < S; ++p) {
      for (int j = 0; j < live; ++j) s[j] += parts[p * n + at + j];
    }
  }
  for (int j = 0; j < live; ++j) store_any(out, type, at + j, s[j]);
}

}  // namespace

// How a product is cut: 128 x 128 tiles, and as many splits of the tokens
// as fill two blocks on each of 256 compute units.
WGradPlan wgrad8_plan(long M, int N, int K, int parts) {
  const int stage = parts == 1 ? 64 : 32;
  WGradPlan p;
  p.tiles_n = ceil_div(N, 128);
  p.tiles_k = ceil_div(K, 128);
  const long stages = (M + stage - 1) / stage;
  const long tiles = (long)p.tiles_n * p.tiles_k;
  long s = 512 / tiles;
  if (s > stages / 4) s = stages / 4;
  if (s < 1) s = 1;
  p.rows = (stages + s - 1) / s * stage;
  p.splits = (int)((M + p.rows - 1) / p.rows);
  if (p.splits < 1) p.splits = 1;
  return p;
}

template <typename TG>
hipError_t wgrad8_t(
    hipStream_t s,
    const TG* g,
    const int8_t* codes,
    const uint8_t* exps,
    long M,
    int N,
    int K,
    const WGradPlan& plan,
    float* parts,  // [splits][N][K]
    float* bias) {  // [splits * tiles_k][N], may be null
  WGrad a{g,    codes, exps, parts, bias, M, N, K, ceil_div(K, kBlock8),
          plan.tiles_n, plan.tiles_k, plan.rows};
  constexpr int NP = sizeof(TG) == 4 ? 3 : std::is_same<TG, __half>::value + 1;
  constexpr int BM = NP == 1 ? 64 : 32;
  const unsigned grid = (unsigned)plan.splits * plan.tiles_n * plan.tiles_k;
  wgrad8_kernel<TG, NP, 128, 128, BM, 2, 2><<<grid, 256, 0, s>>>(a);
  return hipGetLastError();
}

hipError_t wgrad8_add(
    hipStream_t s,
    const float* parts,
    int S,
    long n,
    void* out,
    int type) {
  const long blocks = (n + 1023) / 1024;
  wgrad8_add_kernel<<<(unsigned)blocks, 256, 0, s>>>(parts, S, n, out, type);
  return hipGetLastError();
}

template hipError_t wgrad8_t<float>(
    hipStream_t, const float*, const int8_t*, const uint8_t*, long, int, int,
    const WGradPlan&, float*, float*);
template hipError_t wgrad8_t<__hip_bfloat16>(
    hipStream_t, const __hip_bfloat16*, const int8_t*, const uint8_t*, long,
    int, int, const WGradPlan&, float*, float*);
template hipError_t wgrad8_t<__half>(
    hipStream_t, const __half*, const int8_t*, const uint8_t*, long, int, int,
    const WGradPlan&, float*, float*);

}  // namespace kfac
