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
//
// Measured, whole calls in a row: 16384 tokens x 8192 x 4096 bf16 900 to 930
// us by card (1180 to 1220 TFLOP/s; a product of 8192^3 by the library 1228),
// bound by the clock that the power limit leaves; 16384 x 768 x 2304 74 to 76
// us: 50 in the products, 13 to start, end and write 9 splits' sums, and 12 to
// add these; the same in fp16 159 us, in fp32 197; 8192 x 4096 x 4096 fp32 750
// us (370 TFLOP/s, three times that on the matrix cores).

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
  float* bias;           // [S * bias_tiles][N], may be null
  long M;
  int N, K, blocks;
  int tiles_n, tiles_k;
  int bias_tiles;  // tiles of a row that share the bias's sum
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
// that the four rows of a transposed read lie in different banks. Four rows
// of 32 columns are the 64 banks as they are.
template <int WIDTH>
__device__ __forceinline__ int slot(int r, int c) {
  static_assert(WIDTH == 32 || WIDTH >= 128, "");
  return r * (WIDTH / 8) + (WIDTH == 32 ? c : c ^ ((r & 3) << 2));
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
  constexpr int kG = BM * BN / 8 < kT ? BM * BN / 8 : kT;
  constexpr int GC = BM * BN / 8 / kG;             // chunks a thread, g
  constexpr int XC = BM * BK / 16 / kT;            // 16 codes each
  constexpr int kImage = BM * (NP * BN + BK);      // of one stage
  constexpr int kSteps = BM / 16;
  static_assert(GC * kG * 8 == BM * BN && XC * kT * 16 == BM * BK, "");
  static_assert(kG % (BN / 8) == 0, "a thread keeps its columns");
  __shared__ __attribute__((aligned(16))) short lds[2 * kImage];

  const int tid = threadIdx.x, lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const Tile tile = tile_of(a);
  const int n0 = tile.n * BN, k0 = tile.k * BK;
  const long m0 = tile.split * a.rows;
  const long m1 = m0 + a.rows < a.M ? m0 + a.rows : a.M;
  const int stages = (int)((m1 - m0 + BM - 1) / BM);
  // Leading stages that are read without checks. What a chunk reads behind
  // its row's end are values of the next rows, for columns that nothing is
  // stored of, so these have to be there: 7 and 15 values of them.
  int fast = (int)((m1 - m0) / BM);
  while (fast > 0 && (a.N % 8 != 0 || a.K % 16 != 0)) {
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

  // This thread's pieces of a stage: chunk i of g is kG / (BN / 8) rows
  // below chunk i - 1, and so on. Where g has fewer chunks than there are
  // threads, those behind kG do what the first ones do.
  const int g_row = tid % kG / (BN / 8), g_col = tid % (BN / 8) * 8;
  const int x_row = tid / (BK / 16), x_col = tid % (BK / 16) * 16;
  constexpr int kGDown = kG / (BN / 8), kXDown = kT / (BK / 16);
  // Offsets that differ from lane to lane, next to addresses that do not.
  // A chunk right of the matrix reads the tile's first one instead.
  const int gc = n0 + g_col < a.N ? g_col : 0;
  const int xc = k0 + x_col < a.K ? x_col : 0;
  const unsigned g_at = (unsigned)g_row * a.N + gc;
  const unsigned x_at = (unsigned)x_row * a.K + xc;
  const unsigned e_at = (unsigned)x_row * a.blocks + xc / kBlock8;
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
  constexpr int kQ = kSteps * NP;  // fragments of g and a 16 token step
  static_assert(kSteps % 2 == 0, "fragments alternate");
  bf16x8 f[2][FN], x[2][FK];
  const auto read = [&](const short* gl, int q) {
    const int r = q / NP, p = q % NP;
#pragma unroll
    for (int j = 0; p == 0 && j < FK; ++j) {
      x[r & 1][j] =
          fragment<BK>(gl + NP * BM * BN + x_frag[j] + r * 16 * BK);
    }
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      f[q & 1][i] = fragment<BN>(gl + g_frag[i] + p * BM * BN + r * 16 * BN);
    }
  };
  const auto multiply = [&](int q) {
#pragma unroll
    for (int i = 0; i < FN; ++i) {
#pragma unroll
      for (int j = 0; j < FK; ++j) {
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            f[q & 1][i], x[q / NP & 1][j], acc[i][j], 0, 0, 0);
      }
    }
  };
  // Between two products of a step come a share of its reads, conversions,
  // writes and loads. The two waves of a SIMD leave a barrier together: with
  // all products of a step in a row they would both wait for the matrix core
  // and then both leave it idle (16384 x 8192 x 4096: 954 us, 892 us with
  // this; 2 or 4 reads and 4 to 8 conversions a product are 1 to 10 % slower).
  const auto interleave = [&]() {
#pragma unroll
    for (int i = 0; i < FN * FK; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // matrix product
      __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);  // LDS reads
      __builtin_amdgcn_sched_group_barrier(0x002, 5, 0);  // vector operations
      __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);  // LDS write
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);  // load
    }
  };
  // the first tiles of a row share the work of the bias's sum
  const bool sums_bias = a.bias != nullptr && tile.k < a.bias_tiles;
  const auto add_bias = [&](const short* gl, int stage) {
    if (!sums_bias || stage % a.bias_tiles != tile.k) return;
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
    __syncthreads();
    read(lds, 0);
  }
  for (int stage = 0; stage < fast - 1; ++stage) {
    const short* image = lds + (stage & 1) * kImage;
    short* next = lds + ((stage + 1) & 1) * kImage;
    // in the last turn the last stage is loaded again, and not used
    const int then = stage + 2 < fast ? stage + 2 : fast - 1;
    add_bias(image, stage);
#pragma unroll
    for (int q = 0; q < kQ - 1; ++q) {
      // Before the products of a step come the reads of the next one, behind
      // them a share of the next stage, whose registers take the stage
      // after that.
      read(image, q + 1);
      multiply(q);
#pragma unroll
      for (int i = q * GC / (kQ - 1); i < (q + 1) * GC / (kQ - 1); ++i) {
        put_g(i, next);
        load_g(i, then);
      }
#pragma unroll
      for (int i = q * XC / (kQ - 1); i < (q + 1) * XC / (kQ - 1); ++i) {
        put_x(i, next + NP * BM * BN);
        load_x(i, then);
      }
      interleave();
    }
    // The last step's fragments are in registers: the image is done with,
    // and the next one whole behind the barrier, so that its first
    // fragments are read before these products as well.
    __syncthreads();
    read(next, 0);
    multiply(kQ - 1);
    interleave();
  }
  const auto load_end = [&](int stage) {
    const long m = m0 + (long)stage * BM;
#pragma unroll
    for (int i = 0; i < GC; ++i) {
      const long row = m + g_row + i * kGDown;
      const long left = (a.M - row) * a.N - (n0 + gc);
      gv[i].clear();
      if (row < m1) {
        gv[i].load((const TG*)a.g + row * a.N + n0 + gc, left);
      }
    }
#pragma unroll
    for (int i = 0; i < XC; ++i) {
      const long row = m + x_row + i * kXDown;
      const long left = (a.M - row) * a.K - (k0 + xc);
      const int8_t* p = a.codes + row * a.K + k0 + xc;
      xv[i] = (u32x4)(0u);
      xe[i] = 1;
      if (row < m1) {
        xe[i] = a.exps[row * a.blocks + (k0 + xc) / kBlock8];
        if (left >= 16) {
          xv[i] = load16(p);
        } else {
#pragma unroll
          for (int j = 0; j < 15; ++j) {
            if (j < left) xv[i][j / 4] |= (unsigned)(uint8_t)p[j] << j % 4 * 8;
          }
        }
      }
    }
  };
  // The last whole stage, whose image is there, and the end of the tokens:
  // rows behind it are zero, and what a chunk reads behind its row's end may
  // be missing.
  for (int stage = fast > 0 ? fast - 1 : 0; stage < stages; ++stage) {
    const short* image = lds;
    if (stage < fast) {
      image += (stage & 1) * kImage;
    } else {
      load_end(stage);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < GC; ++i) put_g(i, lds);
#pragma unroll
      for (int i = 0; i < XC; ++i) put_x(i, lds + NP * BM * BN);
      __syncthreads();
      read(lds, 0);
    }
    add_bias(image, stage);
#pragma unroll
    for (int q = 0; q < kQ; ++q) {
      if (q + 1 < kQ) read(image, q + 1);
      multiply(q);
    }
  }

  // column lane % 32, rows 8 * (r / 4) + 4 * (lane / 32) + r % 4
  float* out = a.out + (long)tile.split * a.N * a.K;
  if (n0 + BN <= a.N && k0 + BK <= a.K) {
    // A row's address is the same for a wave: 3 operations a store, not 10
    // (0.8 us of 128 x 128 values, not 1.8).
    float* first = out + (long)(n0 + wn) * a.K + k0 + wk;
    const unsigned at = (unsigned)(lane / 32 * 4) * a.K + lane % 32;
#pragma unroll
    for (int i = 0; i < FN; ++i) {
#pragma unroll
      for (int j = 0; j < FK; ++j) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int n = i * 32 + r / 4 * 8 + r % 4;
          *lane_ptr(first + (long)n * a.K + j * 32, at) = acc[i][j][r];
        }
      }
    }
  } else {
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
  }
  if (sums_bias) {
    // the threads that share columns, added in their order
    float* part = (float*)lds;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (tid < kG) part[g_row * BN + g_col + j] = bias[j];
    }
    __syncthreads();
    for (int c = tid; c < BN; c += kT) {
      float s = 0.f;
      for (int i = 0; i < kGDown; ++i) s += part[i * BN + c];
      if (n0 + c < a.N) {
        a.bias[((long)tile.split * a.bias_tiles + tile.k) * a.N + n0 + c] = s;
      }
    }
  }
}

// One sum over rows: out[i] = sum over r < rows of parts[r][i], i < n. A
// block's 256 threads take 4 columns each, in `groups` that each take every
// groups-th row: a thread waits for each few rows that it reads, and there
// are up to some 30 of the weight's sum, a few hundred of the bias's.
struct Sum {
  const float* parts;
  void* out;
  long n;
  int rows;
  int type;
  int groups;
  unsigned blocks;
};

// Two sums in a launch, the weight's in the first blocks, the bias's behind
// them. The loads of a thread's kTurn rows are under way together: 9 rows of
// 768 x 2304 take 12 us, 14 with 8 and then 1.
constexpr int kTurn = 12;
__global__ __launch_bounds__(256) void wgrad8_add_kernel(
    Sum weight,
    Sum bias) {
  __shared__ float lds[1024];
  const bool second = blockIdx.x >= weight.blocks;
  const Sum a = second ? bias : weight;
  const unsigned block = blockIdx.x - (second ? weight.blocks : 0);
  const int lanes = 256 / a.groups, columns = lanes * 4;
  const int group = threadIdx.x / lanes, lane = threadIdx.x % lanes;
  for (long first = (long)block * columns; first < a.n;
       first += (long)a.blocks * columns) {
    const long at = first + lane * 4;
    const int live = a.n - at < 4 ? (int)(a.n - at) : 4;
    float s[4] = {};
    if (live == 4) {
      for (int r0 = group; r0 < a.rows; r0 += kTurn * a.groups) {
        float v[kTurn][4];
#pragma unroll
        for (int i = 0; i < kTurn; ++i) {
          const int r = r0 + i * a.groups;
          v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.f;
          if (r < a.rows) __builtin_memcpy(v[i], a.parts + r * a.n + at, 16);
        }
#pragma unroll
        for (int i = 0; i < kTurn; ++i) {
#pragma unroll
          for (int j = 0; j < 4; ++j) s[j] += v[i][j];
        }
      }
    } else {
#pragma unroll 4
      for (int r = group; r < a.rows; r += a.groups) {
#pragma unroll
        for (int j = 0; j < 3; ++j) {
          if (j < live) s[j] += a.parts[r * a.n + at + j];
        }
      }
    }
    if (a.groups == 1) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j < live) store_any(a.out, a.type, at + j, s[j]);
      }
      continue;
    }
    __syncthreads();  // the sums of the turn before have been read
#pragma unroll
    for (int j = 0; j < 4; ++j) lds[group * columns + lane * 4 + j] = s[j];
    __syncthreads();
    for (int c = threadIdx.x; c < columns; c += 256) {
      if (first + c >= a.n) break;
      float sum = 0.f;
      for (int i = 0; i < a.groups; ++i) sum += lds[i * columns + c];
      store_any(a.out, a.type, first + c, sum);
    }
  }
}

}  // namespace

// bf16 numbers that a gradient is the sum of.
template <typename TG>
constexpr int kParts =
    sizeof(TG) == 4 ? 3 : std::is_same<TG, __half>::value ? 2 : 1;

// The tiles of a product: small, large, and for up to 64 outputs narrow ones.
// Two images are 128 KB of LDS for large bf16 tiles, one block to a compute
// unit, and 80 KB or less for the others, two blocks or three.
enum Tiles { kSmall, kLarge, kNarrow };

template <typename TG, int TILES>
struct Cut {
  static constexpr int NP = kParts<TG>;
  static constexpr int BN =
      TILES == kNarrow ? 32 : TILES == kLarge && NP == 1 ? 256 : 128;
  static constexpr int BK = TILES == kSmall ? 128 : 256;
  static constexpr int BM = NP == 1 ? 64 : 32;
  static constexpr int WN = TILES == kNarrow ? 1 : 2;
  static constexpr int WK = TILES == kSmall ? 2 : 4;
  static constexpr int kSlots =
      TILES == kNarrow && NP > 1 ? 3 : TILES == kLarge && NP == 1 ? 1 : 2;
};

// What a call takes, in us, by a model with the numbers of 40 shapes on
// MI355X (rows 64 to 16384, widths 64 to 6144, each with some 20 splits;
// the model is within 12 to 14 %, its choice 5 to 8 % from the best):
// a block takes 8 to 10 us beside its stages, a stage the longer the fuller
// the compute unit. Small tiles need more reads for each product (a stage
// of a quarter of the area takes 1.2 us for two blocks, not 0.95), but
// leave less to be added where the tokens are split. Narrow tiles multiply no
// padding where there are few outputs (16384 x 32 x 4096: bf16 25 us, 30 with
// small tiles; fp32 32 us, 61; 64 outputs fp32 48 us, 72; of 96 nothing is
// gained). Few inputs gain little, since a wide gradient is what is read.
struct Rates {
  float alone[3], full[3];  // a stage with half a card's blocks and with all
  float block;
  float add;       // a second launch
  float per_byte;  // of the splits' sums, written and read
  float per_row;   // of them
};

template <typename TG>
constexpr Rates kRates = kParts<TG> == 1
    ? Rates{{0.73f, 1.65f, 0.8f}, {1.22f, 1.89f, 1.6f}, 10.4f, 2.8f, 1.05e-7f, 0.06f}
    : kParts<TG> == 2
    ? Rates{{0.67f, 0.83f, 0.55f}, {1.00f, 2.14f, 1.2f}, 8.1f, 3.8f, 1.37e-7f, 0.06f}
    : Rates{{0.91f, 1.17f, 0.9f}, {1.55f, 3.09f, 1.76f}, 8.6f, 3.2f, 1.36e-7f, 0.07f};

template <typename TG, int TILES>
void consider(long M, int N, int K, WGradPlan& best, float& best_time) {
  using C = Cut<TG, TILES>;
  constexpr Rates rates = kRates<TG>;
  constexpr int kSlots = 256 * C::kSlots;
  const long tiles_n = ceil_div(N, C::BN), tiles_k = ceil_div(K, C::BK);
  const long tiles = tiles_n * tiles_k;
  const long stages = (M + C::BM - 1) / C::BM;
  long last = 0;
  for (const int blocks : {0, 64, 128, 192, 256, 384, 512, 768}) {
    long s = (blocks + tiles / 2) / tiles;
    s = s < 1 ? 1 : s > stages ? stages : s;
    const long per = (stages + s - 1) / s;
    s = (stages + per - 1) / per;
    if (s == last) continue;
    last = s;
    const long all = s * tiles, left = all % kSlots;
    float time = (float)(all / kSlots) *
        (rates.block + (float)per * rates.full[TILES]);
    if (left > 0) {
      // from half a block for each compute unit to all of its blocks
      float load = ((float)left / 256.f - 0.5f) / (C::kSlots - 0.5f);
      load = load < 0.f ? 0.f : load;
      time += rates.block +
          (float)per *
              (rates.alone[TILES] +
               load * (rates.full[TILES] - rates.alone[TILES]));
    }
    if (s > 1) {
      time += rates.add + (float)s * rates.per_row +
          (float)(s * N) * (float)K * 8.f * rates.per_byte;
    }
    if (time < best_time) {
      best_time = time;
      // One tile does the bias's sum alone where that saves the second
      // launch: some 10 % of its stages against 2.5 us.
      const bool alone = s == 1 && per <= 16;
      const long share = alone ? 1 : per < tiles_k ? per : tiles_k;
      best = {TILES, (int)s, (int)tiles_n, (int)tiles_k, (int)share,
              per * C::BM};
    }
  }
}

template <typename TG>
WGradPlan wgrad8_plan(long M, int N, int K) {
  WGradPlan best{};
  float time = __builtin_inff();
  consider<TG, kSmall>(M, N, K, best, time);
  consider<TG, kLarge>(M, N, K, best, time);
  if (N <= 64) consider<TG, kNarrow>(M, N, K, best, time);
  return best;
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
  WGrad a{g,    codes, exps, sums, bias, M, N, K, ceil_div(K, kBlock8),
          plan.tiles_n, plan.tiles_k, plan.bias_tiles, plan.rows};
  const unsigned grid = (unsigned)plan.splits * plan.tiles_n * plan.tiles_k;
  const auto go = [&](auto tiles) {
    using C = Cut<TG, decltype(tiles)::value>;
    wgrad8_kernel<TG, C::NP, C::BN, C::BK, C::BM, C::WN, C::WK>
        <<<grid, C::WN * C::WK * kWave, 0, s>>>(a);
    return hipGetLastError();
  };
  return plan.tiles == kSmall ? go(std::integral_constant<int, kSmall>())
      : plan.tiles == kLarge  ? go(std::integral_constant<int, kLarge>())
                              : go(std::integral_constant<int, kNarrow>());
}

hipError_t wgrad8_add(
    hipStream_t s,
    const float* sums,
    int splits,
    long n,
    void* out,
    int type,
    const float* bias_sums,
    int bias_rows,
    long bias_n,
    void* bias_out,
    int bias_type) {
  const auto sum_of = [](
      const float* parts, void* o, long n, int rows, int type) {
    Sum a{parts, o, o == nullptr ? 0 : n, rows, type, 1, 0};
    // kTurn rows a thread at most, and two blocks for each compute unit as long
    // as a thread has 2 rows or more
    while (a.groups < 32 &&
           (a.groups * kTurn < rows ||
            (a.n * a.groups < 512L * 1024 && a.groups * 4 <= rows))) {
      a.groups *= 2;
    }
    const long columns = 1024 / a.groups;
    const long need = (a.n + columns - 1) / columns;
    a.blocks = (unsigned)(need < (1 << 20) ? need : 1 << 20);
    return a;
  };
  const Sum weight = sum_of(sums, out, n, splits, type);
  const Sum bias =
      sum_of(bias_sums, bias_out, bias_n, bias_rows, bias_type);
  if (weight.blocks + bias.blocks == 0) return hipSuccess;
  wgrad8_add_kernel<<<weight.blocks + bias.blocks, 256, 0, s>>>(weight, bias);
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
