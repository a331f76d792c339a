// Shared by the selective scan's and the causal convolution's kernels: element conversion,
// the functions of the gate and of the step size, sequence ends in packed rows, and the
// fixed-order sum of per-block partials.
#pragma once

#include <initializer_list>
#include <type_traits>

#include "capi_common.cuh"
#include "common.cuh"

namespace ttt {
namespace scan {

template <typename T>
__device__ __forceinline__ float to_f(T x) {
  if constexpr (std::is_same<T, float>::value) return x;
  else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __bfloat162float(x);
  else return __half2float(x);
}
template <typename T>
__device__ __forceinline__ T from_f(float x) {
  if constexpr (std::is_same<T, float>::value) return x;
  else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __float2bfloat16_rn(x);
  else return __float2half_rn(x);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 1 / (1 + e^-x): two special-function operations, a few steps of 2^-23 off.
__device__ __forceinline__ float sigmoid(float x) { return rcp(1.f + ex2(-kLog2e * x)); }
// log(1 + e^x) = max(x, 0) + log(1 + w), w = e^-|x|, by log(1 + w) = 2 artanh(s), s = w / (2 + w)
// <= 1/3, and a polynomial in s^2 for 2 artanh(s) / s (least maximum error 8e-9): relative
// accuracy also where w is small, which a logarithm of 1 + w would lose.
__device__ __forceinline__ float softplus(float x) {
  const float w = ex2(-kLog2e * fabsf(x)), s = w * rcp(2.f + w), v = s * s;
  float q = fmaf(v, 0.2814132571220398f, 0.2797023057937622f);
  q = fmaf(v, q, 0.4002406597137451f);
  q = fmaf(v, q, 0.666663408279419f);
  q = fmaf(v, q, 2.f);
  return fmaf(s, q, fmaxf(x, 0.f));
}
// Packed rows: seq[t] is the sequence that token t belongs to, -1 for tokens of none. A token
// whose predecessor belongs to another sequence starts its own, and likewise at the end.
__device__ __forceinline__ bool seq_starts(const int* seq, int t) { return t == 0 || seq[t] != seq[t - 1]; }
__device__ __forceinline__ bool seq_ends(const int* seq, int t, int T) { return t + 1 >= T || seq[t] != seq[t + 1]; }

// Whether this row's slot may be used: 1, 0 for a row without one (a negative index), -1 for
// an index past the last slot or one that an earlier row has already. Called by all threads.
__device__ __forceinline__ int slot_state(const int* index, int row, int slots) {
  if (!index) return 1;
  const int q = index[row];
  int again = 0;
  for (int r = threadIdx.x; r < row; r += blockDim.x) again |= index[r] == q;
  again = __syncthreads_or(again);
  return q < 0 ? 0 : q >= slots || again ? -1 : 1;
}

// out[w] = sum over m of part[m][w], in one fixed order: 32 columns x 16 row groups a block.
int column_sum(const float* part, long long M, long long W, float* out, cudaStream_t st, const char* who);

inline int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) {
    cudaGetLastError();  // no device here (sizes are asked for on a machine without one)
    return 148;
  }
  return n;
}

}  // namespace scan
}  // namespace ttt
