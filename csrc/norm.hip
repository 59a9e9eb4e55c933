// Layer norm of the rows of a matrix, forward and backward.
//
//   t = round(x + r)            the residual stream, kept in x's type
//   h = (t - mean(t)) * rstd    rstd = 1 / sqrt(mean((t - mean)^2) + eps)
//   y = round(h * w + b)
//
//   q  = dy * w
//   dx = round(rstd * (q - mean(q) - h * mean(q * h)) + dt)
//   dw = sum over rows of dy * h,   db = sum over rows of dy
//
// Both passes are bound by memory, so a row is read once: it stays in
// registers between its sums and its outputs, 8 values a lane and chunk, 8, 16
// or 32 lanes a row up to 64, 128 or 256 values, one wave up to 1024, 4, 8 or
// 16 up to 2048, 4096 or 16384 (the forward pass by half for lengths that are
// no multiple of 8). The variance is the mean of the centred squares of those
// registers, never a difference of two large sums. The backward pass keeps dw
// and db of its rows in registers too and writes one partial row a block; a
// second kernel adds them in a fixed order, so that the gradients are the same
// from run to run. Rows longer than 16384 (or shorter than 8) take the kernels
// at the end of the file, which read a row once for each of its sums.
//
// Measured, whole calls in a row: forward 16384 x 8192 bf16 102 us (5.2 TB/s),
// 16384 x 768 fp32 and a bf16 residual to bf16 and two 8 bit forms 34 us (5.2
// TB/s); backward 150 us (5.4 TB/s) and, from 8 bits, 29 us (4.7 TB/s), with
// some 5 us of each for the parameters' sums. A copy of 1 GiB reaches 5.2
// TB/s.

#include "act8.h"

namespace kfac {

namespace {

template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
  return v + __int_as_float(__builtin_amdgcn_mov_dpp(
                 __float_as_int(v), CTRL, 0xf, 0xf, true));
}

// v of the lane and of the one 16 (32) further, round the wave
__device__ __forceinline__ float add_swap16(float v) {
  const unsigned u = __float_as_uint(v);
  const auto row = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return __uint_as_float(row[0]) + __uint_as_float(row[1]);
}
__device__ __forceinline__ float add_swap32(float v) {
  const unsigned u = __float_as_uint(v);
  const auto half = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(half[0]) + __uint_as_float(half[1]);
}

// Sum over each 8, 16, 32 or 64 lanes, the same bits in all of them: quads,
// halves and rows of 16 by register permutations, rows and halves of the
// wave by swaps.
template <int LANES>
__device__ __forceinline__ float lane_sum(float v) {
  v = add_dpp<0xB1>(v);
  v = add_dpp<0x4E>(v);
  v = add_dpp<0x141>(v);
  if (LANES >= 16) v = add_dpp<0x140>(v);
  if (LANES >= 32) v = add_swap16(v);
  if (LANES >= 64) v = add_swap32(v);
  return v;
}

// Sum over the lanes of a wave that are LANES, 2 * LANES ... apart.
template <int LANES>
__device__ __forceinline__ float sum_across(float v) {
  if (LANES <= 8) v = add_dpp<0x128>(v);  // a row of 16 turned by 8
  if (LANES <= 16) v = add_swap16(v);
  if (LANES <= 32) v = add_swap32(v);
  return v;
}

// Sum over the LANES of a row: part of a wave, or several waves, whose blocks
// call it with all of them, as often as each other. `at` alternates between
// two halves of `lds`, so that one barrier a sum is enough.
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* lds, int& at) {
  constexpr int W = LANES / kWave;
  v = lane_sum<W == 0 ? LANES : kWave>(v);
  if (W <= 1) return v;
  const int wave = threadIdx.x / kWave;
  float* slot = lds + at * 16;
  at ^= 1;
  if (threadIdx.x % kWave == 0) slot[wave] = v;
  __syncthreads();
  const int first = wave / W * W;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) s += slot[first + i];
  return s;
}

// 1 / sqrt(v), a Newton step behind the instruction's 1 ulp: a row's values
// share this error, and where they round to 16 bits it decides for all.
__device__ __forceinline__ float reciprocal_root(float v) {
  const float r = rsqrtf(v);
  const float left = fmaf(-v * r, r, 1.f);
  // no step from or to 0 and infinity
  return fabsf(left) < 1.f ? fmaf(0.5f * r, left, r) : r;
}

struct Param {
  const void* p;  // may be null
  int type;
};

// 8 values from start + at on; the lanes of a wave share `start`.
__device__ __forceinline__ void load_any(
    const Param& a,
    long start,
    unsigned at,
    float v[8]) {
  if (a.type == kF32) {
    load8(lane_ptr((const float*)a.p + start, at), v);
  } else if (a.type == kBF16) {
    load8(lane_ptr((const __hip_bfloat16*)a.p + start, at), v);
  } else {
    load8(lane_ptr((const __half*)a.p + start, at), v);
  }
}

template <typename TX, typename TY>
struct Forward {
  const TX* x;
  Param r, w, b;
  TX* total;  // written if r is there
  TY* y;
  float* mean;
  float* rstd;
  int8_t* in_codes;  // may be null
  uint8_t* in_exps;
  int8_t* out_codes;  // may be null
  uint8_t* out_exps;
  long R;
  int D;
  int blocks;  // exponents a row
  float eps;
};

// Rows of up to 64, 128 and 256 values take 8, 16 and 32 lanes, so that a
// wave has 8, 4 or 2 of them: rows_of_wave. Its first row's number is in a
// scalar register (wide rows have one for each of their waves), and addresses
// cost no vector registers: the others are some 32 bit offset further down.
// Where there are no more rows, lanes repeat the first one, to the bit. These
// kernels are bound by arithmetic where lanes are idle: 196608 rows of 64 bf16
// values take 10 us forward and 17 backward, 51 and 56 with a wave a row.
constexpr int rows_of_wave(int lanes) {
  return lanes < kWave ? kWave / lanes : 1;
}
template <int LANES>
__device__ __forceinline__ int group_of() {
  constexpr int threads = LANES < kWave ? kWave : LANES;
  return __builtin_amdgcn_readfirstlane(threadIdx.x / threads) *
      rows_of_wave(LANES);
}
// The lane's row, counted from the wave's first, of which there are `left`.
template <int LANES>
__device__ __forceinline__ int down_of(long left) {
  if (LANES >= kWave) return 0;
  const int down = threadIdx.x % kWave / LANES;
  return down < left ? down : 0;
}

// The part of a row that a lane holds in chunk i of its NCH: 8 values from
// `col`, of which those from `skip` on are its own. Where a row's length is
// no multiple of 8 (ODD, 9 or more), the last lane takes the row's last 8
// values, and its neighbour owns the first of them: both compute the same
// results for these, and only sums have to leave one out.
struct Part {
  int chunk;
  unsigned col;
  unsigned at;  // the column, from the start of the wave's first row
  int skip;
  bool any;
};

template <bool ODD, int LANES, int NCH>
__device__ __forceinline__ Part part_of(int lane, int i, int D, int down = 0) {
  Part p;
  p.chunk = lane + i * LANES;
  const int col = p.chunk * kChunk;
  // rows reach into the last of a lane's chunks, see by_width
  const bool whole = i + 1 < NCH;
  p.any = whole || col < D;
  p.skip = ODD && !whole && p.any && col > D - kChunk ? col - (D - kChunk) : 0;
  p.col = p.any ? col - p.skip : 0;
  p.at = down * D + p.col;
  return p;
}

// How many of the columns that a wave's last chunks of a row cover are in it:
// span_of or more if all are, 0 or less if the wave is right of its end.
constexpr int span_of(int lanes) {
  return (lanes < kWave ? lanes : kWave) * kChunk;
}
template <int LANES, int NCH>
__device__ __forceinline__ int columns_of(int D) {
  const int wave =
      LANES <= kWave ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  return D - (NCH - 1) * LANES * kChunk - wave * kWave * kChunk;
}

// The lane's number, new to the compiler in each turn of a loop: it would
// keep a 64 bit address a lane for each tensor otherwise, and spill.
__device__ __forceinline__ int fresh(int lane) {
  asm volatile("" : "+v"(lane));
  return lane;
}

template <typename TX, typename TY, int NCH, int LANES, bool ODD>
__global__ __launch_bounds__(
    LANES <= kWave ? 256 : LANES) void norm_fwd_kernel(
    Forward<TX, TY> a) {
  constexpr int G = LANES <= kWave ? 4 * rows_of_wave(LANES) : 1;  // of a block
  __shared__ float lds[32];
  int at = 0;
  const int lane0 = threadIdx.x % LANES;
  const int group = group_of<LANES>();
  float w[NCH][8], b[NCH][8];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const Part p = part_of<ODD, LANES, NCH>(lane0, i, a.D);
#pragma unroll
    for (int j = 0; j < kChunk; ++j) w[i][j] = 1.f, b[i][j] = 0.f;
    if (a.w.p != nullptr) load_any(a.w, 0, p.col, w[i]);
    if (a.b.p != nullptr) load_any(a.b, 0, p.col, b[i]);
  }
  const int columns = columns_of<LANES, NCH>(a.D);
  for (long base = (long)blockIdx.x * G; base < a.R;
       base += (long)gridDim.x * G) {
    const long row = base + group;
    if (LANES <= kWave && row >= a.R) return;
    if (NCH == 1 && LANES > kWave && columns <= 0) {
      // right of the row's end: only keeps the others company
      row_sum<LANES>(0.f, lds, at);
      row_sum<LANES>(0.f, lds, at);
      continue;
    }
    const long start = row * a.D;
    const int lane = fresh(lane0);
    const int down = down_of<LANES>(a.R - row);
    float t[NCH][8];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const Part p = part_of<ODD, LANES, NCH>(lane, i, a.D, down);
      load8(lane_ptr(a.x + start, p.at), t[i]);
      if (a.r.p != nullptr) {
        float r[8];
        load_any(a.r, start, p.at, r);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
          t[i][j] = round_to(t[i][j] + r[j], a.x);
        }
        if (p.any) store8(lane_ptr(a.total + start, p.at), t[i]);
      }
      if (i + 1 < NCH || columns >= span_of(LANES)) {
#pragma unroll
        for (int j = 0; j < kChunk; ++j) sum += t[i][j];
      } else {
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
          sum += p.any && j >= p.skip ? t[i][j] : 0.f;
        }
      }
    }
    const float mean = row_sum<LANES>(sum, lds, at) / a.D;
    float square = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const Part p = part_of<ODD, LANES, NCH>(lane, i, a.D, down);
      if (i + 1 < NCH || columns >= span_of(LANES)) {
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
          const float c = t[i][j] - mean;
          square += c * c;
        }
      } else {
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
          const float c = p.any && j >= p.skip ? t[i][j] - mean : 0.f;
          square += c * c;
        }
      }
    }
    const float var = row_sum<LANES>(square, lds, at) / a.D;
    const float rstd = reciprocal_root(var + a.eps);
    if (lane == 0) {
      (a.mean + row)[down] = mean;
      (a.rstd + row)[down] = rstd;
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const Part p = part_of<ODD, LANES, NCH>(lane, i, a.D, down);
      const long block = row * a.blocks;
      if (a.in_codes != nullptr) {
        pack_chunk<ODD>(
            t[i], p.any, p.skip, kChunk, lane_ptr(a.in_codes + start, p.at),
            lane_ptr(a.in_exps + block, down * a.blocks + p.chunk / 8), p.chunk % 8 == 0);
      }
#pragma unroll
      for (int j = 0; j < kChunk; ++j) {
        const float h = (t[i][j] - mean) * rstd;
        t[i][j] = round_to(h * w[i][j] + b[i][j], a.y);
      }
      if (p.any) store8(lane_ptr(a.y + start, p.at), t[i]);
      if (a.out_codes != nullptr) {
        pack_chunk<ODD>(
            t[i], p.any, p.skip, kChunk, lane_ptr(a.out_codes + start, p.at),
            lane_ptr(a.out_exps + block, down * a.blocks + p.chunk / 8), p.chunk % 8 == 0);
      }
    }
  }
}

template <typename TX, typename TY>
struct Backward {
  const TY* dy;
  const TX* x;  // null: codes and exps
  const int8_t* codes;
  const uint8_t* exps;
  const float* mean;
  const float* rstd;
  Param w;
  const TX* dt;  // may be null
  TX* dx;
  float* partial;  // [gridDim.x][2][D], null if no parameter has a gradient
                   // or a single block writes it
  void* dw;        // either may be null
  void* db;
  int dw_type, db_type;
  long R;
  int D;
  int blocks;
};

template <typename TX, typename TY>
__device__ __forceinline__ void load_kept(
    const Backward<TX, TY>& a,
    long row,
    int col,
    int n,
    float v[8]) {
  const long at = row * a.D + col;
  if (a.x != nullptr) {
    load_chunk(a.x + at, n, v);
  } else if (n > 0) {
    const unsigned byte = a.exps[row * a.blocks + col / kBlock8];
    unpack_chunk(a.codes + at, byte, n, v);
  } else {
#pragma unroll
    for (int j = 0; j < kChunk; ++j) v[j] = 0.f;
  }
}

// What the backward pass reads of a row, as it is in memory.
template <typename TX, typename TY, int NCH>
struct KeptRow {
  Raw<TY> dy[NCH];
  Raw<TX> x[NCH];  // or 8 codes in its first 8 bytes
  unsigned byte[NCH], own[NCH];  // exponents
  float mean, rstd;

  template <bool ODD, bool KEPT8, int LANES>
  __device__ __forceinline__ void fetch(
      const Backward<TX, TY>& a,
      long row,
      int lane,
      int down) {
    const long start = row * a.D;
    mean = (a.mean + row)[down];
    rstd = (a.rstd + row)[down];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const Part p = part_of<ODD, LANES, NCH>(lane, i, a.D, down);
      dy[i].load(lane_ptr(a.dy + start, p.at));
      if (KEPT8) {
        const uint8_t* e = a.exps + row * a.blocks;
        byte[i] = *lane_ptr(e, down * a.blocks + p.col / kBlock8);
        // the last lane's own values may be in the next block
        if (ODD) {
          own[i] = *lane_ptr(e, down * a.blocks + (p.any ? p.chunk / 8 : 0));
        }
        unsigned c[2];
        __builtin_memcpy(c, lane_ptr(a.codes + start, p.at), 8);
        x[i].v[0][0] = c[0];
        x[i].v[0][1] = c[1];
      } else {
        x[i].load(lane_ptr(a.x + start, p.at));
      }
    }
  }

  template <bool ODD, bool KEPT8>
  __device__ __forceinline__ void values(int i, const Part& p, float v[8]) {
    if (!KEPT8) {
      x[i].values(v);
      return;
    }
    const float s = scale_of(byte[i]);
    codes4(x[i].v[0][0], s, v);
    codes4(x[i].v[0][1], s, v + 4);
    if (ODD && p.skip > 0) {
      const float t = scale_of(own[i]);
      float w[8];
      codes4(x[i].v[0][0], t, w);
      codes4(x[i].v[0][1], t, w + 4);
#pragma unroll
      for (int j = 0; j < kChunk; ++j) v[j] = j < p.skip ? v[j] : w[j];
    }
  }
};

template <typename TX, typename TY, int NCH, int LANES, bool ODD, bool KEPT8>
__global__ __launch_bounds__(1024) void norm_bwd_kernel(Backward<TX, TY> a) {
  constexpr int S = rows_of_wave(LANES);
  constexpr int G = LANES < kWave ? 16 : 1024 / LANES;  // groups of a block
  constexpr int kAll = LANES * kChunk * NCH;            // columns of a group
  __shared__ float lds[32];
  __shared__ __attribute__((aligned(16))) float
      parts[G > 1 ? 2 * G * kAll : 4];
  int at = 0;
  const int lane0 = threadIdx.x % LANES;
  const int group = group_of<LANES>();  // its first row
  const float mean_of = 1.f / a.D;
  float w[NCH][8], dw[NCH][8], db[NCH][8];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const Part p = part_of<ODD, LANES, NCH>(lane0, i, a.D);
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
      w[i][j] = 1.f;
      dw[i][j] = db[i][j] = 0.f;
    }
    if (a.w.p != nullptr) load_any(a.w, 0, p.col, w[i]);
  }
  // Where a row takes several waves, barriers keep them together, and a
  // row's loads have to be under way before the last row is done with (16384
  // x 8192 bf16: 176 us without, 159 us with it, 5.1 TB/s). Single waves wait
  // for their rows in their own time.
  constexpr bool kAhead = LANES > kWave && NCH == 1;  // two chunks would spill
  KeptRow<TX, TY, NCH> next;
  if (kAhead) {
    const long row = (long)blockIdx.x * G + group;
    next.template fetch<ODD, KEPT8, LANES>(a, row < a.R ? row : 0, lane0, 0);
  }
  for (long base = (long)blockIdx.x * G * S; base < a.R;
       base += (long)gridDim.x * G * S) {
    const bool some = base + group < a.R;
    if (LANES <= kWave && !some) break;
    // a group without a row takes part in the barriers, with row 0
    const long row = some ? base + group : 0;
    const long start = row * a.D;
    const int lane = fresh(lane0);
    const int down = down_of<LANES>(a.R - row);
    const bool live =
        some && (S == 1 || row + (int)threadIdx.x % kWave / LANES < a.R);
    if (!kAhead) next.template fetch<ODD, KEPT8, LANES>(a, row, lane, down);
    const float mean = next.mean, rstd = next.rstd;
    Raw<TY> dy[NCH];
    Raw<TX> dt[NCH];
    float h[NCH][8];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const Part p = part_of<ODD, LANES, NCH>(lane, i, a.D, down);
      dy[i] = next.dy[i];
      next.template values<ODD, KEPT8>(i, p, h[i]);
    }
    if (a.dt != nullptr) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const Part p = part_of<ODD, LANES, NCH>(lane, i, a.D, down);
        dt[i].load(lane_ptr(a.dt + start, p.at));
      }
    } else {
#pragma unroll
      for (int i = 0; i < NCH; ++i) dt[i].clear();
    }
    if (kAhead) {
      const long then = base + (long)gridDim.x * G + group;
      next.template fetch<ODD, KEPT8, LANES>(
          a, then < a.R ? then : 0, lane, 0);
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const Part p = part_of<ODD, LANES, NCH>(lane, i, a.D, down);
      float g[8];
      dy[i].values(g);
#pragma unroll
      for (int j = 0; j < kChunk; ++j) {
        h[i][j] = (h[i][j] - mean) * rstd;
        const float own = live && p.any && j >= p.skip ? g[j] : 0.f;
        const float product = own * h[i][j];
        dw[i][j] += product;
        db[i][j] += own;
        // added here, not behind the stores: both terms would be kept
        asm volatile("" : "+v"(dw[i][j]), "+v"(db[i][j]));
        s1 += own * w[i][j];
        s2 += product * w[i][j];
      }
    }
    s1 = row_sum<LANES>(s1, lds, at) * mean_of;
    s2 = row_sum<LANES>(s2, lds, at) * mean_of;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const Part p = part_of<ODD, LANES, NCH>(lane, i, a.D, down);
      float g[8], d[8];
      dy[i].values(g);
      dt[i].values(d);
#pragma unroll
      for (int j = 0; j < kChunk; ++j) {
        d[j] += rstd * (g[j] * w[i][j] - s1 - h[i][j] * s2);
      }
      if (live && p.any) store8(lane_ptr(a.dx + start, p.at), d);
    }
  }
  // the rows of a wave, in the order of their lanes' permutations
  if (S > 1) {
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
      dw[0][j] = sum_across<LANES>(dw[0][j]);
      db[0][j] = sum_across<LANES>(db[0][j]);
    }
  }
  // a single block's sums are the gradients
  const bool single = a.partial == nullptr;
  if (single && a.dw == nullptr && a.db == nullptr) return;
  const auto put = [&](int which, int col, float v) {
    if (!single) {
      a.partial[((long)blockIdx.x * 2 + which) * a.D + col] = v;
    } else if (which && a.db != nullptr) {
      store_any(a.db, a.db_type, col, v);
    } else if (!which && a.dw != nullptr) {
      store_any(a.dw, a.dw_type, col, v);
    }
  };
  if (G == 1) {
    float* mine = a.partial + (long)blockIdx.x * 2 * a.D;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const Part p = part_of<ODD, LANES, NCH>(lane0, i, a.D);
      if (!p.any) continue;
      if (!single && p.skip == 0) {
        store8(mine + p.col, dw[i]);
        store8(mine + a.D + p.col, db[i]);
        continue;
      }
#pragma unroll
      for (int j = 0; j < kChunk; ++j) {
        if (j >= p.skip) {
          put(0, p.col + j, dw[i][j]);
          put(1, p.col + j, db[i][j]);
        }
      }
    }
    return;
  }
  // The groups' sums, added in the order of the groups. They lie by chunks:
  // the last chunk of an odd row holds its columns from D - 8 on.
  const int last = ODD ? a.D / kChunk * kChunk : a.D;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    float* mine = parts + group / S * kAll + (lane0 + i * LANES) * kChunk;
    if (S > 1 && threadIdx.x % kWave >= LANES) continue;
    store8(mine, dw[i]);
    store8(mine + G * kAll, db[i]);
  }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * a.D; c += 1024) {
    const int which = c >= a.D, col = which ? c - a.D : c;
    const int at = col < last ? col : col + last - (a.D - kChunk);
    float s = 0.f;
#pragma unroll
    for (int g = 0; g < G; ++g) s += parts[(which * G + g) * kAll + at];
    put(which, col, s);
  }
}

// out[c] = sum over P of partial[p][which][c]: 64 columns a block, 16 waves
// that each add every 16th row.
__global__ __launch_bounds__(1024) void norm_param_kernel(
    const float* __restrict__ partial,
    int P,
    int D,
    void* dw,
    int dw_type,
    void* db,
    int db_type) {
  __shared__ float lds[16][kWave];
  const int which = blockIdx.y;
  void* out = which ? db : dw;
  if (out == nullptr) return;
  const int lane = threadIdx.x % kWave;
  const int wave = threadIdx.x / kWave;
  const int c = blockIdx.x * kWave + lane;
  float s = 0.f;
  if (c < D) {
#pragma unroll 4
    for (int p = wave; p < P; p += 16) {
      s += partial[((long)p * 2 + which) * D + c];
    }
  }
  lds[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && c < D) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += lds[i][lane];
    store_any(out, which ? db_type : dw_type, c, s);
  }
}

// -- rows longer than 16384: one block a row, which is read again from
// memory (or the cache) for each of its sums -------------------------------

constexpr int kLongSpan = 1024 * kChunk;

template <typename TX, typename TY>
__global__ __launch_bounds__(1024) void norm_fwd_long_kernel(
    Forward<TX, TY> a) {
  __shared__ float lds[32];
  int at = 0;
  const int first = threadIdx.x * kChunk;
  const TX* kept = a.r.p != nullptr ? a.total : a.x;
  for (long row = blockIdx.x; row < a.R; row += gridDim.x) {
    const long start = row * a.D;
    float sum = 0.f;
    for (int c0 = 0; c0 < a.D; c0 += kLongSpan) {
      const int col = c0 + first, n = a.D - col;
      if (n <= 0) break;
      float t[8];
      load_chunk(a.x + start + col, n, t);
      if (a.r.p != nullptr) {
        float r[8];
        load_chunk(a.r.p, a.r.type, start + col, n, r);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) t[j] = round_to(t[j] + r[j], a.x);
        // read again by the lane that wrote it
        store_chunk(a.total + start + col, n, t);
      }
      float part = 0.f;
#pragma unroll
      for (int j = 0; j < kChunk; ++j) part += t[j];
      sum += part;
    }
    const float mean = row_sum<1024>(sum, lds, at) / a.D;
    float square = 0.f;
    for (int c0 = 0; c0 < a.D; c0 += kLongSpan) {
      const int col = c0 + first, n = a.D - col;
      if (n <= 0) break;
      float t[8], part = 0.f;
      load_chunk(kept + start + col, n, t);
#pragma unroll
      for (int j = 0; j < kChunk; ++j) {
        const float c = j < n ? t[j] - mean : 0.f;
        part += c * c;
      }
      square += part;
    }
    const float var = row_sum<1024>(square, lds, at) / a.D;
    const float rstd = reciprocal_root(var + a.eps);
    if (threadIdx.x == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
    // whole blocks of lanes: pack_chunk compares 8 neighbours
    for (int c0 = 0; c0 < a.D; c0 += kLongSpan) {
      const int col = c0 + first, n = a.D - col;
      const int chunk = col / kChunk;
      const long block = row * a.blocks + chunk / 8;
      float t[8];
      load_chunk(kept + start + col, n, t);
      if (a.in_codes != nullptr) {
        pack_chunk<false>(
            t, n > 0, 0, n, a.in_codes + start + col, a.in_exps + block,
            chunk % 8 == 0);
      }
      float w[8], b[8];
#pragma unroll
      for (int j = 0; j < kChunk; ++j) w[j] = 1.f, b[j] = 0.f;
      if (a.w.p != nullptr) load_chunk(a.w.p, a.w.type, col, n, w);
      if (a.b.p != nullptr) load_chunk(a.b.p, a.b.type, col, n, b);
#pragma unroll
      for (int j = 0; j < kChunk; ++j) {
        t[j] = j < n ? round_to((t[j] - mean) * rstd * w[j] + b[j], a.y) : 0.f;
      }
      store_chunk(a.y + start + col, n, t);
      if (a.out_codes != nullptr) {
        pack_chunk<false>(
            t, n > 0, 0, n, a.out_codes + start + col, a.out_exps + block,
            chunk % 8 == 0);
      }
    }
  }
}

template <typename TX, typename TY>
__global__ __launch_bounds__(1024) void norm_bwd_long_kernel(
    Backward<TX, TY> a) {
  __shared__ float lds[32];
  int at = 0;
  const int first = threadIdx.x * kChunk;
  for (long row = blockIdx.x; row < a.R; row += gridDim.x) {
    const long start = row * a.D;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s1 = 0.f, s2 = 0.f;
    for (int pass = 0; pass < 2; ++pass) {
      for (int c0 = 0; c0 < a.D; c0 += kLongSpan) {
        const int col = c0 + first, n = a.D - col;
        if (n <= 0) break;
        float q[8], h[8], w[8];
        load_chunk(a.dy + start + col, n, q);
        load_kept(a, row, col, n, h);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) w[j] = 1.f;
        if (a.w.p != nullptr) load_chunk(a.w.p, a.w.type, col, n, w);
        float p1 = 0.f, p2 = 0.f;
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
          h[j] = j < n ? (h[j] - mean) * rstd : 0.f;
          q[j] = j < n ? q[j] * w[j] : 0.f;
          p1 += q[j];
          p2 += q[j] * h[j];
        }
        if (pass == 0) {
          s1 += p1;
          s2 += p2;
          continue;
        }
#pragma unroll
        for (int j = 0; j < kChunk; ++j) q[j] = rstd * (q[j] - s1 - h[j] * s2);
        if (a.dt != nullptr) {
          float d[8];
          load_chunk(a.dt + start + col, n, d);
#pragma unroll
          for (int j = 0; j < kChunk; ++j) q[j] += d[j];
        }
        store_chunk(a.dx + start + col, n, q);
      }
      if (pass == 0) {
        s1 = row_sum<1024>(s1, lds, at) / a.D;
        s2 = row_sum<1024>(s2, lds, at) / a.D;
      }
    }
  }
}

// dw and db of long rows: a block takes 2048 columns, 8 a lane, and every
// gridDim.y-th row.
template <typename TX, typename TY>
__global__ __launch_bounds__(256) void norm_bwd_long_param_kernel(
    Backward<TX, TY> a) {
  const int col = (blockIdx.x * 256 + threadIdx.x) * kChunk;
  const int n = a.D - col;
  if (n <= 0) return;
  float dw[8] = {}, db[8] = {};
  for (long row = blockIdx.y; row < a.R; row += gridDim.y) {
    const float mean = a.mean[row], rstd = a.rstd[row];
    float q[8], h[8];
    load_chunk(a.dy + row * a.D + col, n, q);
    load_kept(a, row, col, n, h);
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
      dw[j] += j < n ? q[j] * ((h[j] - mean) * rstd) : 0.f;
      db[j] += q[j];
    }
  }
  float* mine = a.partial + (long)blockIdx.y * 2 * a.D;
  store_chunk(mine + col, n, dw);
  store_chunk(mine + a.D + col, n, db);
}

// 16 waves x 2 chunks of 8 a lane. Rows of 1 to 7 values, of which no lane
// can take 8, go the way of the longer ones too.
bool is_long(int D) { return D > 16384 || D < kChunk; }
constexpr int kLongSplit = 128;  // partial rows of the long form
unsigned long_blocks(long R) { return (unsigned)(R < 65536 ? R : 65536); }

// Blocks of the backward kernel: what fills 256 compute units once, each
// with the 16 waves that 128 registers a lane allow.
int rows_of_block(int D) {
  return D <= 64 ? 128
      : D <= 128  ? 64
      : D <= 256  ? 32
      : D <= 1024 ? 16
      : D <= 2048 ? 4
      : D <= 4096 ? 2
                  : 1;
}

// Calls fn with the kernel's template parameters (chunks of a lane, waves of
// a row, odd length) as types. Rows reach into the last chunk: part_of counts
// on that. With HALVED the rows of odd lengths take half the waves and two
// chunks a lane where they would take 4 to 16 waves: they start at any
// alignment, such loads take longer, and more of these rows are under way at
// a time. Forward, 46 M values of bf16 in rows of 1025, 1501, 2047, 3001, 4095,
// 5001, 6697 and 8191: 64, 49, 41, 50, 43, 63, 51 and 45 us halved, 79, 56, 47,
// 63, 53, 84, 72 and 65 not; fp32 1 to 19 % less halved. Rows of 6696 take 42
// us and 41, and 57 to 60 with an 8 bit form: even rows keep one chunk.
// Backward, the other way about: 75, 61, 56, 62, 58, 82, 73 and 71 us with one
// chunk, 88, 70, 60, 71, 64, 80, 72 and 68 with two, fp32 all slower by 1 to 9
// %, since two chunks leave no registers for the next row's loads.
template <bool HALVED, typename Fn>
hipError_t by_width(int D, Fn fn) {
  const auto go = [&](auto odd) {
    constexpr int kHalf = HALVED && decltype(odd)::value ? 2 : 1;
    const auto call = [&](auto nch, auto lanes) { return fn(nch, lanes, odd); };
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using Chunks = std::integral_constant<int, kHalf>;
    return D <= 64  ? call(I1(), std::integral_constant<int, 8>())
        : D <= 128  ? call(I1(), std::integral_constant<int, 16>())
        : D <= 256  ? call(I1(), std::integral_constant<int, 32>())
        : D <= 512  ? call(I1(), std::integral_constant<int, 64>())
        : D <= 1024 ? call(I2(), std::integral_constant<int, 64>())
        : D <= 2048 ? call(Chunks(), std::integral_constant<int, 256 / kHalf>())
        : D <= 4096 ? call(Chunks(), std::integral_constant<int, 512 / kHalf>())
        : D <= 8192
        ? call(Chunks(), std::integral_constant<int, 1024 / kHalf>())
        : call(I2(), std::integral_constant<int, 1024>());
  };
  return D % kChunk ? go(std::true_type()) : go(std::false_type());
}

}  // namespace

// Blocks of the backward pass. A few turns are left to a single block, which
// then writes the gradients itself: a second launch takes 2 to 3 us, a turn 1
// us of up to 512 values, 1.7 of 1024 and 3.5 of 8192.
static int norm_bwd_blocks(long R, int D) {
  if (is_long(D)) return (int)(R < kLongSplit ? R : kLongSplit);
  const long need = (R + rows_of_block(D) - 1) / rows_of_block(D);
  if (need <= (D <= 512 ? 4 : D <= 4096 ? 2 : 1)) return 1;
  const long turns = (need + 255) / 256;  // the same for each block
  return (int)((need + turns - 1) / turns);
}

int norm_bwd_partials(long R, int D) {
  const int blocks = norm_bwd_blocks(R, D);
  return blocks == 1 && !is_long(D) ? 0 : blocks;
}

template <typename TX, typename TY>
hipError_t norm_fwd_t(
    hipStream_t s,
    const TX* x,
    const void* r,
    int r_type,
    const void* w,
    int w_type,
    const void* b,
    int b_type,
    TX* total,
    TY* y,
    float* mean,
    float* rstd,
    int8_t* in_codes,
    uint8_t* in_exps,
    int8_t* out_codes,
    uint8_t* out_exps,
    long R,
    int D,
    float eps) {
  Forward<TX, TY> a{x,        {r, r_type}, {w, w_type}, {b, b_type},
                    total,    y,           mean,        rstd,
                    in_codes, in_exps,     out_codes,   out_exps,
                    R,        D,           ceil_div(D, kBlock8), eps};
  if (is_long(D)) {
    norm_fwd_long_kernel<TX, TY><<<long_blocks(R), 1024, 0, s>>>(a);
    return hipGetLastError();
  }
  // 8 waves a SIMD: 2048 blocks of 256 threads, 512 of 1024
  return by_width<true>(D, [&](auto nch, auto lanes, auto odd) {
    constexpr int N = decltype(nch)::value, L = decltype(lanes)::value;
    constexpr int threads = L <= kWave ? 256 : L;
    constexpr int rows = L <= kWave ? 4 * rows_of_wave(L) : 1;
    const long need = (R + rows - 1) / rows;
    const long most = 2048L * 256 / threads;
    norm_fwd_kernel<TX, TY, N, L, decltype(odd)::value>
        <<<(unsigned)(need < most ? need : most), threads, 0, s>>>(a);
    return hipGetLastError();
  });
}

template <typename TX, typename TY>
hipError_t norm_bwd_t(
    hipStream_t s,
    const TY* dy,
    const TX* x,
    const int8_t* codes,
    const uint8_t* exps,
    const float* mean,
    const float* rstd,
    const void* w,
    int w_type,
    const TX* dt,
    TX* dx,
    float* partial,
    void* dw,
    int dw_type,
    void* db,
    int db_type,
    long R,
    int D) {
  Backward<TX, TY> a{dy, x,       codes, exps, mean,    rstd,    {w, w_type},
                     dt, dx,      partial, dw, db,      dw_type, db_type,
                     R,  D,       ceil_div(D, kBlock8)};
  const int P = norm_bwd_blocks(R, D);
  if (is_long(D)) {
    norm_bwd_long_kernel<TX, TY><<<long_blocks(R), 1024, 0, s>>>(a);
    KFAC_HIP_CHECK(hipGetLastError());
    if (partial != nullptr) {
      const dim3 grid(ceil_div(D, 256 * kChunk), P);
      norm_bwd_long_param_kernel<TX, TY><<<grid, 256, 0, s>>>(a);
      KFAC_HIP_CHECK(hipGetLastError());
    }
  } else {
    KFAC_HIP_CHECK(by_width<false>(D, [&](auto nch, auto lanes, auto odd) {
      constexpr int N = decltype(nch)::value, L = decltype(lanes)::value;
      constexpr bool ODD = decltype(odd)::value;
      if (x != nullptr) {
        norm_bwd_kernel<TX, TY, N, L, ODD, false><<<P, 1024, 0, s>>>(a);
      } else {
        norm_bwd_kernel<TX, TY, N, L, ODD, true><<<P, 1024, 0, s>>>(a);
      }
      return hipGetLastError();
    }));
  }
  if (partial == nullptr) return hipSuccess;
  norm_param_kernel<<<dim3(ceil_div(D, kWave), 2), 1024, 0, s>>>(
      partial, P, D, dw, dw_type, db, db_type);
  return hipGetLastError();
}

#define KFAC_NORM(TX, TY)                                                     \
  template hipError_t norm_fwd_t<TX, TY>(                                     \
      hipStream_t, const TX*, const void*, int, const void*, int,             \
      const void*, int, TX*, TY*, float*, float*, int8_t*, uint8_t*, int8_t*, \
      uint8_t*, long, int, float);                                            \
  template hipError_t norm_bwd_t<TX, TY>(                                     \
      hipStream_t, const TY*, const TX*, const int8_t*, const uint8_t*,       \
      const float*, const float*, const void*, int, const TX*, TX*, float*,   \
      void*, int, void*, int, long, int);
KFAC_NORM(float, float)
KFAC_NORM(float, __hip_bfloat16)
KFAC_NORM(float, __half)
KFAC_NORM(__hip_bfloat16, __hip_bfloat16)
KFAC_NORM(__hip_bfloat16, float)
KFAC_NORM(__half, __half)
KFAC_NORM(__half, float)
#undef KFAC_NORM

}  // namespace kfac
