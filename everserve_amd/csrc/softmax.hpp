// What the attention kernels share: vector types, sums over lanes, and a row's running softmax.
#pragma once

#include "common.hpp"

namespace evs {

constexpr float kLn2 = 0.6931471805599453f;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

// A value that all lanes have alike, as a scalar.
__device__ __forceinline__ unsigned long long scalar(unsigned long long v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
  return static_cast<unsigned long long>(hi) << 32 | lo;
}

// The lane's number, afresh: what is computed from it is computed in every part, where the compiler
// would move it ahead of all parts and keep it in registers that the stages need.
__device__ __forceinline__ int lane_now() {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  return lane;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  bf16x2 v;
  v[0] = static_cast<__bf16>(lo);
  v[1] = static_cast<__bf16>(hi);
  return __builtin_bit_cast(uint32_t, v);
}

__device__ __forceinline__ float across_rows_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}

__device__ __forceinline__ float across_rows_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// A value at a device address that is a multiple of four; an address out of LDS must say so, or the
// load counts as one that may be of LDS and is waited for with those.
template <typename T>
__device__ __forceinline__ T load_global(uint64_t p) {
  typedef T Packed __attribute__((aligned(4)));
  return *reinterpret_cast<const __attribute__((address_space(1))) Packed*>(p);
}

// ---------------------------------------------------------------- softmax
// The reference that a row's weights are taken against may lag its maximum by this much (in
// powers of two): the sums are only rescaled when some row's maximum has grown past it. (Weights
// are up to 2^8 then, so a mean of V above 2^119 may pass f32 on its way.)
constexpr float kSlack = 8.0f;

// A row's running state: four lanes hold the same m and shift, and a part of the sum l each.
struct Running {
  float m = -INFINITY, l = 0.0f;

  // What the weights are taken against; a row may have seen nothing yet.
  __device__ __forceinline__ float shift() const { return m == -INFINITY ? 0.0f : m; }
};

// The scores of tokens that a row does not see, and of those that are none, masked: `ahead` is the
// number of tokens from this lane's first of the 32 up to the row's last, `ok` has a bit a token.
template <int kTiles>
__device__ __forceinline__ void mask(float (&s)[kTiles][8], const int (&ahead)[kTiles],
                                     uint32_t ok) {
#pragma unroll
  for (int k = 0; k < 8; k++) {
    const int at = 16 * (k >> 2) + (k & 3);
    const bool in = (ok >> at) & 1;
#pragma unroll
    for (int n = 0; n < kTiles; n++) s[n][k] = ahead[n] >= at && in ? s[n][k] : -INFINITY;
  }
}

// Whether new scores of each of this lane's rows (masked ones -infinity) take some row's maximum too
// far past its reference: then all sums so far must be multiplied by `fade`.
template <int kTiles, int kScores>
__device__ __forceinline__ bool grow(const float (&s)[kTiles][kScores], float scale_log2,
                                     Running (&r)[kTiles], float (&fade)[kTiles]) {
  float top[kTiles];
  bool far = false;
#pragma unroll
  for (int n = 0; n < kTiles; n++) {
    float x = s[n][0];
#pragma unroll
    for (int k = 1; k < kScores; k++) x = fmaxf(x, s[n][k]);
    top[n] = x * scale_log2;
    far |= top[n] > r[n].m + kSlack;
  }
  if (__builtin_amdgcn_ballot_w64(far) == 0) return false;
#pragma unroll
  for (int n = 0; n < kTiles; n++) {
    const float m = fmaxf(across_rows_max(top[n]), r[n].m);
    const float before = r[n].m;
    r[n].m = m;
    fade[n] = __builtin_amdgcn_exp2f(before - r[n].shift());
    r[n].l *= fade[n];
  }
  return true;
}

}  // namespace evs
