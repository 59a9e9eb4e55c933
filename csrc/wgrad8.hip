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

struct Tile {
  int split, n, k;
};

// Block -> tile. Blocks go to the 8 dies in turn, each with a cache of its
// own: a die gets consecutive tiles, which share a split's tokens, and its
// 32 compute units a patch of 8 x 4 tiles, which read 5 bytes of memory a
// token for each 24 that they use (256 x 256 tiles).
__device__ __forceinline__ Tile tile_of(const WGrad& a) {
  const int total = gridDim.x, die = blockIdx.x % 8, each = total / 8;
  const int extra = total % 8;
  int i = die * each + (die < extra ? die : extra) + blockIdx.x / 8;
  const int tiles = a.tiles_n * a.tiles_k;
  const int split = i / tiles;
  i -= split * tiles;
  const int strip = i / (8 * a.tiles_k);
  const int high =
      a.tiles_n - strip * 8 < 8 ? a.tiles_n - strip * 8 : 8;
  i -= strip * 8 * a.tiles_k;
  return {split, strip * 8 + i % high, i / high};
}

// 16 byte chunk c of row r: the 64 byte group is swapped by the row, so
// that the four rows of a transposed read lie in different banks.
template <int WIDTH>
__device__ __forceinline__ int slot(int r, int c) {
  return r * (WIDTH / 8) + (c ^ ((r & 3) << 2));
}

// Where a lane's part of the fragment of 32 columns starts: its 8 tokens are
// 8 * (lane / 32) + j, its column is lane % 32. The read gives each of 16
// lanes 4 tokens of one of 16 columns, and takes from each the address of 4
// columns of one token. Tokens 4 and 16 further down are at fixed distances.
template <int WIDTH>
__device__ __forceinline__ int fragment_at(int col, int lane) {
  const int i = lane % 16;
  const int c = col + lane / 16 % 2 * 16 + i % 4 * 4;
  return slot<WIDTH>(lane / 32 * 8 + i / 4, c / 8) * 8 + c % 8;
}
template <int WIDTH>
__device__ __forceinline__ bf16x8 fragment(const short* at) {
  typedef __attribute__((address_space(3))) short4v* Ptr;
  const short4v a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)at);
  const short4v b =
      __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(at + 4 * WIDTH));
  typedef __attribute__((ext_vector_type(8))) short short8v;
  const short8v v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_bit_cast(bf16x8, v);
}

__device__ __forceinline__ unsigned high_halves(float lo, float hi) {
  // bytes 2, 3 of both: exact, since the values have 8 bits or fewer
  return __builtin_amdgcn_perm(
      __float_as_uint(hi), __float_as_uint(lo), 0x07060302);
}

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
  constexpr int kSteps = BM / 16;
  static_assert(GC * kT * 8 == BM * BN && XC * kT * 16 == BM * BK, "");
  static_assert(kT % (BN / 8) == 0, "a thread keeps its columns");
  __shared__ __attribute__((aligned(16))) short lds[2 * kImage];

  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const Tile tile = tile_of(a);
  const int n0 = tile.n * BN, k0 = tile.k * BK;
  const long m0 = tile.split * a.rows;
  const long m1 = m0 + a.rows < a.M ? m0 + a.rows : a.M;
  const int stages = (int)((m1 - m0 + BM - 1) / BM);
  // Leading stages that are read without checks. What a chunk reads behind
  // its row's end are values of the next rows, for columns that nothing is
  // stored of, so these have to be there: 7 and 15 values of them.
  int fast = (int)((m1 - m0) / BM);
  while (fast > 0) {
    const long rest = a.M - m0 - (long)fast * BM;
    if (rest * a.N >= 7 && rest * a.K >= 15) break;
    --fast;
  }

  f32x16 acc[FN][FK];
#pragma unroll
  for (int i = 0; i < FN; ++i) {
#pragma unroll
    for (int j = 0; j < FK; ++j) acc[i][j] = (f32x16)(0.f);
  }
  float bias[8] = {};

  // This thread's pieces of a stage: chunk i of g is kT / (BN / 8) rows
  // below chunk i - 1, and so on.
  const int g_row = tid / (BN / 8), g_col = tid % (BN / 8) * 8;
  const int x_row = tid / (BK / 16), x_col = tid % (BK / 16) * 16;
  constexpr int kGDown = kT / (BN / 8), kXDown = kT / (BK / 16);
  // Offsets that differ from lane to lane, next to addresses that do not.
  // A chunk right of the matrix reads the tile's first one instead.
  const int gc = n0 + g_col < a.N ? g_col : 0;
  const int xc = k0 + x_col < a.K ? x_col : 0;
  const unsigned g_at = g_row * a.N + gc, x_at = x_row * a.K + xc;
  const unsigned e_at = x_row * a.blocks + xc / kBlock8;
  Raw<TG> gv[GC];
  u32x4 xv[XC];
  unsigned xe[XC];
  const auto load_g = [&](int i, int stage) {
    const long m = m0 + (long)stage * BM + i * kGDown;
    gv[i].load((const TG*)a.g + m * a.N + n0 + g_at);
  };
  const auto load_x = [&](int i, int stage) {
    const long m = m0 + (long)stage * BM + i * kXDown;
    xv[i] = load16(a.codes + m * a.K + k0 + x_at);
    xe[i] = (a.exps + m * a.blocks + k0 / kBlock8)[e_at];
  };
  const auto put_g = [&](int i, short* gl) {
    const int at = slot<BN>(g_row + i * kGDown, g_col / 8) * 8;
    if (NP == 1) {
      __builtin_memcpy(gl + at, &gv[i].v[0], 16);
      return;
    }
    float v[8];
    gv[i].values(v);
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      unsigned part[4];
      take_part(v, part);
      __builtin_memcpy(gl + p * BM * BN + at, part, 16);
    }
  };
  const auto put_x = [&](int i, short* xl) {
    const float s = scale_of(xe[i]);
    unsigned v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float f[4];
      codes4(xv[i][j], s, f);
      v[2 * j] = high_halves(f[0], f[1]);
      v[2 * j + 1] = high_halves(f[2], f[3]);
    }
    const int row = x_row + i * kXDown, chunk = x_col / 8;
    __builtin_memcpy(xl + slot<BK>(row, chunk) * 8, v, 16);
    __builtin_memcpy(xl + slot<BK>(row, chunk + 1) * 8, v + 4, 16);
  };

  const int wn = wave / WK * TN, wk = wave % WK * TK;
  int g_frag[FN], x_frag[FK];
#pragma unroll
  for (int i = 0; i < FN; ++i) g_frag[i] = fragment_at<BN>(wn + i * 32, lane);
#pragma unroll
  for (int j = 0; j < FK; ++j) x_frag[j] = fragment_at<BK>(wk + j * 32, lane);
  // The products of a stage's image; other(r) runs between them.
  const auto products = [&](const short* gl, int stage, auto other) {
    const short* xl = gl + NP * BM * BN;
    if (a.bias != nullptr && stage % a.tiles_k == tile.k) {
      // the tiles of a row share the work of the bias's sum
#pragma unroll
      for (int i = 0; i < GC * NP; ++i) {
        const int row = g_row + i % GC * kGDown;
        float v[8];
        load8(
            (const __hip_bfloat16*)gl + i / GC * BM * BN +
                slot<BN>(row, g_col / 8) * 8,
            v);
#pragma unroll
        for (int j = 0; j < 8; ++j) bias[j] += v[j];
      }
    }
    // the next step's fragments are read before this step's products, which
    // hide the read
    bf16x8 f[2][FN], x[2][FK];
    const auto read = [&](int q) {
      const int r = q / NP, p = q % NP;
#pragma unroll
      for (int j = 0; p == 0 && j < FK; ++j) {
        x[r & 1][j] = fragment<BK>(xl + x_frag[j] + r * 16 * BK);
      }
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        f[q & 1][i] =
            fragment<BN>(gl + g_frag[i] + p * BM * BN + r * 16 * BN);
      }
    };
    read(0);
#pragma unroll
    for (int q = 0; q < kSteps * NP; ++q) {
      if (q + 1 < kSteps * NP) read(q + 1);
#pragma unroll
      for (int i = 0; i < FN; ++i) {
#pragma unroll
        for (int j = 0; j < FK; ++j) {
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              f[q & 1][i], x[q / NP & 1][j], acc[i][j], 0, 0, 0);
        }
      }
      if (q % NP == NP - 1) other(q / NP);
    }
  };

  if (fast > 0) {
    const int second = fast > 1 ? 1 : 0;
#pragma unroll
    for (int i = 0; i < GC; ++i) load_g(i, 0);
#pragma unroll
    for (int i = 0; i < XC; ++i) load_x(i, 0);
#pragma unroll
    for (int i = 0; i < GC; ++i) {
      put_g(i, lds);
      load_g(i, second);
    }
#pragma unroll
    for (int i = 0; i < XC; ++i) {
      put_x(i, lds + NP * BM * BN);
      load_x(i, second);
    }
  }
  for (int stage = 0; stage < fast; ++stage) {
    __syncthreads();
    short* next = lds + ((stage + 1) & 1) * kImage;
    // past the end the last stage is loaded again, and not used
    const int then = stage + 2 < fast ? stage + 2 : fast - 1;
    products(lds + (stage & 1) * kImage, stage, [&](int r) {
      // a share of the next stage goes to LDS while the products run, and
      // its registers take the stage after that
#pragma unroll
      for (int i = r * GC / kSteps; i < (r + 1) * GC / kSteps; ++i) {
        put_g(i, next);
        load_g(i, then);
      }
#pragma unroll
      for (int i = r * XC / kSteps; i < (r + 1) * XC / kSteps; ++i) {
        put_x(i, next + NP * BM * BN);
        load_x(i, then);
      }
    });
  }
  for (int stage = fast; stage < stages; ++stage) {
    // the end of the tokens: every value is checked
    const long m = m0 + (long)stage * BM;
    __syncthreads();
#pragma unroll 1
    for (int c = tid; c < BM * BN / 8; c += kT) {
      const int row = c / (BN / 8), col = c % (BN / 8) * 8;
      float v[8];
      load_chunk(
          (const TG*)a.g + (m + row) * a.N + n0 + col,
          m + row < m1 ? a.N - n0 - col : 0, v);
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        unsigned part[4];
        take_part(v, part);
        __builtin_memcpy(
            lds + p * BM * BN + slot<BN>(row, col / 8) * 8, part, 16);
      }
    }
#pragma unroll 1
    for (int c = tid; c < BM * BK / 8; c += kT) {
      const int row = c / (BK / 8), col = c % (BK / 8) * 8;
      const int n = m + row < m1 ? a.K - k0 - col : 0;
      float v[8] = {};
      if (n > 0) {
        const long at = (m + row) * a.K + k0 + col;
        unpack_chunk(
            a.codes + at,
            a.exps[(m + row) * a.blocks + (k0 + col) / kBlock8], n, v);
      }
      unsigned h[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = high_halves(v[2 * j], v[2 * j + 1]);
      __builtin_memcpy(
          lds + NP * BM * BN + slot<BK>(row, col / 8) * 8, h, 16);
    }
    __syncthreads();
    products(lds, stage, [](int) {});
  }

  // column lane % 32, rows 8 * (r / 4) + 4 * (lane / 32) + r % 4
  float* out = a.out + (long)tile.split * a.N * a.K;
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
    float* part = (float*)lds;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) part[g_row * BN + g_col + j] = bias[j];
    __syncthreads();
    for (int c = tid; c < BN; c += kT) {
      float s = 0.f;
      for (int i = 0; i < kGDown; ++i) s += part[i * BN + c];
      if (n0 + c < a.N) {
        a.bias[((long)tile.split * a.tiles_k + tile.k) * a.N + n0 + c] = s;
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

// Tiles of 256 x 256 with 64 tokens a stage for bf16 gradients, 128 x 256
// with 32 for those that are split: two images are 128 KB and 80 or 64 KB
// of LDS.
template <typename TG>
struct Cut {
  static constexpr int NP =
      sizeof(TG) == 4 ? 3 : std::is_same<TG, __half>::value ? 2 : 1;
  static constexpr int BN = NP == 1 ? 256 : 128, BK = 256;
  static constexpr int BM = NP == 1 ? 64 : 32;
};

template <typename TG>
WGradPlan wgrad8_plan(long M, int N, int K) {
  using C = Cut<TG>;
  WGradPlan p;
  p.tiles_n = ceil_div(N, C::BN);
  p.tiles_k = ceil_div(K, C::BK);
  const long stages = (M + C::BM - 1) / C::BM;
  const long tiles = (long)p.tiles_n * p.tiles_k;
  long s = 256 / tiles;
  if (s > stages / 4) s = stages / 4;
  if (s < 1) s = 1;
  p.rows = (stages + s - 1) / s * C::BM;
  p.splits = (int)((M + p.rows - 1) / p.rows);
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
    float* sums,
    float* bias) {
  using C = Cut<TG>;
  WGrad a{g,    codes, exps, sums, bias, M, N, K, ceil_div(K, kBlock8),
          plan.tiles_n, plan.tiles_k, plan.rows};
  const unsigned grid = (unsigned)plan.splits * plan.tiles_n * plan.tiles_k;
  wgrad8_kernel<TG, C::NP, C::BN, C::BK, C::BM, 2, 4>
      <<<grid, 512, 0, s>>>(a);
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

#define KFAC_WGRAD8(TG)                                                       \
  template WGradPlan wgrad8_plan<TG>(long, int, int);                         \
  template hipError_t wgrad8_t<TG>(                                           \
      hipStream_t, const TG*, const int8_t*, const uint8_t*, long, int, int,  \
      const WGradPlan&, float*, float*);
KFAC_WGRAD8(float)
KFAC_WGRAD8(__hip_bfloat16)
KFAC_WGRAD8(__half)
#undef KFAC_WGRAD8

}  // namespace kfac
