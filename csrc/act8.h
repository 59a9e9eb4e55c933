// Device helpers of the kernels that keep a transformer block's
// activations in 8 bits (norm.hip, act8.hip, wgrad8.hip).
//
// The 8 bit form of a row: blocks of 64 consecutive values share one power
// of two 2^e, the least with max |x| <= 127 * 2^e, and a value is stored as
// the integer nearest to x / 2^e (ties to even). A power of two makes the
// scaling and the way back exact, and code * 2^e has 7 significant bits, so
// it is exact in bf16 too: the only rounding is the one to the code.
// The exponent byte holds e + 127. It lies in [1, 248]: 2^-126 is the
// least normal number, and 127 * 2^121 is the largest multiple that fp32
// holds (larger values saturate to it). 255 marks a block with a NaN or an
// infinity, all of which reads back as NaN.
#pragma once

#include <type_traits>

#include "common.h"
#include "training.h"

namespace kfac {

constexpr int kChunk = 8;    // values that a lane holds: 8 lanes a block

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

// 8 consecutive values. memcpy, because rows of an odd width start at any
// multiple of the element: gfx950 loads and stores 16 bytes there as well.
__device__ __forceinline__ void load8(const float* p, float v[8]) {
  __builtin_memcpy(v, p, 32);
}
__device__ __forceinline__ void load8(const __hip_bfloat16* p, float v[8]) {
  bf16x8 t;
  __builtin_memcpy(&t, p, 16);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (float)t[j];
}
__device__ __forceinline__ void load8(const __half* p, float v[8]) {
  f16x8 t;
  __builtin_memcpy(&t, p, 16);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (float)t[j];
}

__device__ __forceinline__ void store8(float* p, const float v[8]) {
  __builtin_memcpy(p, v, 32);
}
__device__ __forceinline__ void store8(__hip_bfloat16* p, const float v[8]) {
  bf16x8 t;
#pragma unroll
  for (int j = 0; j < 8; ++j) t[j] = (__bf16)v[j];
  __builtin_memcpy(p, &t, 16);
}
__device__ __forceinline__ void store8(__half* p, const float v[8]) {
  f16x8 t;
#pragma unroll
  for (int j = 0; j < 8; ++j) t[j] = (_Float16)v[j];
  __builtin_memcpy(p, &t, 16);
}

__device__ __forceinline__ float round_to(float v, const float*) { return v; }
__device__ __forceinline__ float round_to(float v, const __hip_bfloat16*) {
  return (float)(__bf16)v;
}
__device__ __forceinline__ float round_to(float v, const __half*) {
  return (float)(_Float16)v;
}

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __hip_bfloat16* p) {
  return (float)*(const __bf16*)p;
}
__device__ __forceinline__ float load1(const __half* p) {
  return (float)*(const _Float16*)p;
}
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__hip_bfloat16* p, float v) {
  *(__bf16*)p = (__bf16)v;
}
__device__ __forceinline__ void store1(__half* p, float v) {
  *(_Float16*)p = (_Float16)v;
}

typedef __attribute__((ext_vector_type(4))) unsigned u32x4;

__device__ __forceinline__ u32x4 load16(const void* p) {
  u32x4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}

// 8 values as they are in memory, for loads long before their use.
template <typename T>
struct Raw {
  u32x4 v[sizeof(T) / 2];

  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = load16(p + i * 4);
  }
  // The same where only the first `left` may be there; v is clear.
  __device__ __forceinline__ void load(const T* p, long left) {
    if (left >= kChunk) {
      load(p);
      return;
    }
#pragma unroll
    for (int j = 0; j < kChunk - 1; ++j) {
      if (j >= left) continue;
      if (sizeof(T) == 4) {
        unsigned w;
        __builtin_memcpy(&w, p + j, 4);
        v[j * sizeof(T) / 16][j % 4] = w;
      } else {
        unsigned short h;
        __builtin_memcpy(&h, p + j, 2);
        v[0][j / 2] |= (unsigned)h << j % 2 * 16;
      }
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = (u32x4)(0u);
  }
  __device__ __forceinline__ void values(float f[8]) const {
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
      const unsigned w = v[j * sizeof(T) / 16][j * sizeof(T) / 4 % 4];
      if (sizeof(T) == 4) {
        f[j] = __uint_as_float(w);
      } else if (std::is_same<T, __hip_bfloat16>::value) {
        f[j] = __uint_as_float(j % 2 ? w & 0xFFFF0000 : w << 16);
      } else {
        const unsigned short h = (unsigned short)(w >> j % 2 * 16);
        f[j] = (float)__builtin_bit_cast(_Float16, h);
      }
    }
  }
};

// base[at]: a 32 bit offset of a lane next to an address that its wave
// shares, which is kept in scalar registers.
template <typename T>
__device__ __forceinline__ T* lane_ptr(T* base, unsigned at) {
  using Byte = std::conditional_t<std::is_const<T>::value, const char, char>;
  return (T*)((Byte*)base + at * (unsigned)sizeof(T));
}

// n of 8 values (n <= 0: none); the others read as 0 and are not written.
template <typename T>
__device__ __forceinline__ void load_chunk(const T* p, int n, float v[8]) {
  if (n >= kChunk) {
    load8(p, v);
  } else {
#pragma unroll
    for (int j = 0; j < kChunk; ++j) v[j] = j < n ? load1(p + j) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store_chunk(T* p, int n, const float v[8]) {
  if (n >= kChunk) {
    store8(p, v);
  } else {
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
      if (j < n) store1(p + j, v[j]);
    }
  }
}

__device__ __forceinline__ void load_chunk(
    const void* p,
    int type,
    long at,
    int n,
    float v[8]) {
  if (type == kF32) {
    load_chunk((const float*)p + at, n, v);
  } else if (type == kBF16) {
    load_chunk((const __hip_bfloat16*)p + at, n, v);
  } else {
    load_chunk((const __half*)p + at, n, v);
  }
}
__device__ __forceinline__ void store_any(
    void* p,
    int type,
    long at,
    float v) {
  if (type == kF32) {
    store1((float*)p + at, v);
  } else if (type == kBF16) {
    store1((__hip_bfloat16*)p + at, v);
  } else {
    store1((__half*)p + at, v);
  }
}

// Maximum over the 8 lanes of a block: two quad permutations and a
// reversal of each half row, register moves without a trip through LDS.
__device__ __forceinline__ unsigned max_of_block(unsigned m) {
  unsigned o = __builtin_amdgcn_mov_dpp(m, 0xB1, 0xf, 0xf, true);
  m = m > o ? m : o;
  o = __builtin_amdgcn_mov_dpp(m, 0x4E, 0xf, 0xf, true);
  m = m > o ? m : o;
  o = __builtin_amdgcn_mov_dpp(m, 0x141, 0xf, 0xf, true);
  return m > o ? m : o;
}

// Exponent byte of a block from the bits of max |x|. The bits order like
// the numbers, infinities and NaN above all.
__device__ __forceinline__ unsigned exponent_of(unsigned top) {
  const unsigned p = top >> 23;
  if (p == 255) return 255;
  // 127 * 2^e = 1.984375 * 2^(e+6), whose mantissa bits are 0x7E0000
  const int b = (int)p - 6 + ((top & 0x7FFFFF) > 0x7E0000 ? 1 : 0);
  return b < 1 ? 1 : (b > 248 ? 248 : b);
}

__device__ __forceinline__ float scale_of(unsigned byte) {
  return __uint_as_float(byte == 255 ? 0x7FC00000u : byte << 23);
}

// Code B of the four in a word, as a float: one instruction.
template <int B>
__device__ __forceinline__ float code(unsigned word) {
  float v;
  if (B == 0) {
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD "
        "src0_sel:BYTE_0" : "=v"(v) : "v"(word));
  } else if (B == 1) {
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD "
        "src0_sel:BYTE_1" : "=v"(v) : "v"(word));
  } else if (B == 2) {
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD "
        "src0_sel:BYTE_2" : "=v"(v) : "v"(word));
  } else {
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD "
        "src0_sel:BYTE_3" : "=v"(v) : "v"(word));
  }
  return v;
}

__device__ __forceinline__ void codes4(unsigned word, float s, float v[4]) {
  v[0] = code<0>(word) * s;
  v[1] = code<1>(word) * s;
  v[2] = code<2>(word) * s;
  v[3] = code<3>(word) * s;
}

// max(|a|, |b|, |c|), NaN if one is: one instruction.
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float v;
  asm("v_maximum3_f32 %0, |%1|, |%2|, |%3|"
      : "=v"(v)
      : "v"(a), "v"(b), "v"(c));
  return v;
}

// Packs the 8 values of each lane; all lanes of a block take part. Only the
// values from `skip` on belong to the block (0 unless PART), and none unless
// `any`: the others are not looked at, and their codes not written. Of a row
// that ends inside the lane's 8 the first n are written, behind them are
// zeros.
template <bool PART>
__device__ __forceinline__ void pack_chunk(
    const float v[8],
    bool any,
    int skip,
    int n,
    int8_t* codes,
    uint8_t* exponent,
    bool first) {
  float m[8];
#pragma unroll
  for (int j = 0; j < kChunk; ++j) m[j] = PART && j < skip ? 0.f : v[j];
  float top = max3_abs(m[0], m[1], m[2]);
  top = max3_abs(top, m[3], m[4]);
  top = max3_abs(top, m[5], m[6]);
  top = max3_abs(top, m[7], m[7]);
  const unsigned byte =
      exponent_of(max_of_block(any ? __float_as_uint(top) : 0));
  if (!any) return;
  // 2^-e; a block that holds no number gets codes of 0
  const float inv = __uint_as_float(byte == 255 ? 0u : (254 - byte) << 23);
  if (byte == 248) {
    // the one exponent that is bounded from above: 127 * 2^121
    const float most = __uint_as_float(0x7F7E0000);
    asm volatile("");  // a branch, not 8 operations for everyone
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
      m[j] = __builtin_amdgcn_fmed3f(m[j], -most, most);
    }
  }
  // The fma rounds to an integer (1.5 * 2^23 is even: ties go to even) whose
  // low byte is the code.
  unsigned q[8], c[2];
#pragma unroll
  for (int j = 0; j < kChunk; ++j) {
    q[j] = __float_as_uint(fmaf(m[j], inv, 12582912.f));
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const unsigned lo =
        __builtin_amdgcn_perm(q[4 * j + 1], q[4 * j], 0x0C0C0400);
    const unsigned hi =
        __builtin_amdgcn_perm(q[4 * j + 3], q[4 * j + 2], 0x04000C0C);
    c[j] = byte == 255 ? 0 : lo | hi;
  }
  if ((!PART || skip == 0) && n >= kChunk) {
    __builtin_memcpy(codes, c, 8);
  } else {
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
      if ((!PART || j >= skip) && j < n) {
        codes[j] = (int8_t)(c[j / 4] >> j % 4 * 8);
      }
    }
  }
  if (first) *exponent = (uint8_t)byte;
}

__device__ __forceinline__ void unpack8(
    const int8_t* codes,
    unsigned byte,
    float v[8]) {
  const float s = scale_of(byte);
  unsigned c[2];
  __builtin_memcpy(c, codes, 8);
  codes4(c[0], s, v);
  codes4(c[1], s, v + 4);
}

__device__ __forceinline__ void unpack_chunk(
    const int8_t* codes,
    unsigned byte,
    int n,
    float v[8]) {
  if (n >= kChunk) {
    unpack8(codes, byte, v);
  } else {
    const float s = scale_of(byte);
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
      v[j] = j < n ? (float)codes[j] * s : 0.f;
    }
  }
}

}  // namespace kfac
