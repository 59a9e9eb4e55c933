// Host entry points of the transformer block's training kernels (norm.hip,
// act8.hip, wgrad8.hip), for their binding in training.cpp.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>

namespace kfac {

// Types that are known at launch only (weights, residual branches).
enum DType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

constexpr int kBlock8 = 64;  // values of a row that share an exponent

template <typename T>
hipError_t pack8_t(
    hipStream_t, const T* x, int8_t* codes, uint8_t* exps, long R, int D);
template <typename T>
hipError_t unpack8_t(
    hipStream_t, const int8_t* codes, const uint8_t* exps, T* out, long R,
    int D);
// codes and exps may be null, of both or either
template <typename T>
hipError_t gelu8_fwd_t(
    hipStream_t, const T* x, T* y, int8_t* in_codes, uint8_t* in_exps,
    int8_t* out_codes, uint8_t* out_exps, long R, int D, bool tanh);
template <typename T>
hipError_t gelu8_bwd_t(
    hipStream_t, const T* dy, const int8_t* codes, const uint8_t* exps,
    T* dx, long R, int D, bool tanh);

// r, w, b, total, *_codes and *_exps may be null; total is written if r is
// there
template <typename TX, typename TY>
hipError_t norm_fwd_t(
    hipStream_t, const TX* x, const void* r, int r_type, const void* w,
    int w_type, const void* b, int b_type, TX* total, TY* y, float* mean,
    float* rstd, int8_t* in_codes, uint8_t* in_exps, int8_t* out_codes,
    uint8_t* out_exps, long R, int D, float eps);
// rows of the workspace that the backward pass sums the parameters'
// gradients in, which may be 0
int norm_bwd_partials(long R, int D);
// x or (codes, exps); w, dt, dw, db may be null. partial holds
// norm_bwd_partials(R, D) x 2 x D floats, or is null if that is 0 or there
// is neither dw nor db.
template <typename TX, typename TY>
hipError_t norm_bwd_t(
    hipStream_t, const TY* dy, const TX* x, const int8_t* codes,
    const uint8_t* exps, const float* mean, const float* rstd, const void* w,
    int w_type, const TX* dt, TX* dx, float* partial, void* dw, int dw_type,
    void* db, int db_type, long R, int D);

// How a weight gradient is cut into blocks.
struct WGradPlan {
  int tiles;             // small, large or narrow ones
  int splits;            // of the tokens
  int tiles_n, tiles_k;  // of the output
  int bias_tiles;        // of a row, which share the bias's sum
  long rows;             // tokens of a split
};
template <typename TG>
WGradPlan wgrad8_plan(long M, int N, int K);
// sums: [splits][N][K]; bias: [splits * bias_tiles][N], may be null
template <typename TG>
hipError_t wgrad8_t(
    hipStream_t, const TG* g, const int8_t* codes, const uint8_t* exps,
    long M, int N, int K, const WGradPlan& plan, float* sums, float* bias);
// out[i] = sum over s < splits of sums[s][i], i < n, and the same for the
// bias; either output may be null
hipError_t wgrad8_add(
    hipStream_t, const float* sums, int splits, long n, void* out,
    int type, const float* bias_sums, int bias_rows, long bias_n,
    void* bias_out, int bias_type);

}  // namespace kfac
