// The 4-bit half-rows of a paged cache, shared by the kernels that write, read and attend over
// them (fp4.hip, attend.hip).
//
// A half-row is the K or the V of one slot and head, d elements (d a multiple of 8, 16 to 256):
//   d / 2 bytes of E2M1 codes, element j in bits 4 (j % 8) of dword j / 8;
//   one byte for each 32 elements, the power of two 2^(byte - 127) their codes are multiplied
//   with (an E8M0 scale; 255: the group holds no number and reads as NaN);
//   zeros up to a multiple of 4 bytes.
// These are the operands of gfx950's scaled conversions, which turn two codes and a scale into two
// bf16 or f32 values in one full-rate instruction (132 lane-operations per ns and CU measured, as
// an FMA), exactly: a code times a power of two has two significant bits. (Some codes times 2^126
// or 2^127 are past f32 and bf16, and become infinities; no write makes those scales.)
#pragma once

#include "common.hpp"

namespace evs {

constexpr int kFp4Group = 32;     // elements that share a scale
constexpr int kFp4MinDim = 16;
constexpr int kFp4MaxDim = 256;
constexpr int kScaleNaN = 255;

inline int64_t fp4_groups(int64_t d) { return (d + kFp4Group - 1) / kFp4Group; }
inline int64_t fp4_row_bytes(int64_t d) { return (d / 2 + fp4_groups(d) + 3) / 4 * 4; }

// Element types of full-width rows, queries and outputs (EVS_BF16, EVS_F16, EVS_F32).
inline int64_t elem_bytes(int type) { return type == EVS_F32 ? 4 : 2; }

// A 4-bit cache as its kernels address it: strides in bytes.
struct Fp4Cache {
  char* base;
  int64_t sb, so, sh, skv;  // page, slot in page, head, K to V
  int32_t num_blocks, block_size;
  FastDiv div_bs;
  bool slots32;  // every slot id is below 2^31, div_bs's range
  int32_t heads, d;
  int32_t W;   // dwords of codes in a half-row
  int32_t NG;  // scale bytes in it
};

// Fill `c` after checking that the kernels can address the cache as described; EVS_OK, or an error
// with its message set.
inline int fp4_cache(const char* who, const void* cache, int64_t num_blocks, int64_t block_size,
                     int64_t heads, int64_t d, const int64_t* strides, Fp4Cache& c) {
  EVS_REQUIRE(d >= kFp4MinDim && d <= kFp4MaxDim && d % 8 == 0,
              "%s: head size %lld: a multiple of 8 from %d to %d", who, static_cast<long long>(d),
              kFp4MinDim, kFp4MaxDim);
  EVS_REQUIRE(strides != nullptr, "%s: a layout is five strides", who);
  EVS_REQUIRE(num_blocks >= 0 && num_blocks < (int64_t{1} << 31) && block_size > 0 &&
                  block_size < (int64_t{1} << 31) && heads > 0 && heads < (int64_t{1} << 16),
              "%s: bad cache: %lld pages of %lld slots and %lld heads", who,
              static_cast<long long>(num_blocks), static_cast<long long>(block_size),
              static_cast<long long>(heads));
  EVS_REQUIRE(strides[4] == 1, "%s: a half-row's bytes must be contiguous (element stride %lld)",
              who, static_cast<long long>(strides[4]));
  EVS_REQUIRE(cache != nullptr || num_blocks == 0, "%s: null cache", who);
  bool aligned = (reinterpret_cast<uintptr_t>(cache) & 3) == 0;
  for (int i = 0; i < 4; i++) aligned = aligned && (strides[i] & 3) == 0;
  EVS_REQUIRE(aligned, "%s: the cache and its strides must be multiples of 4 bytes", who);
  c.base = static_cast<char*>(const_cast<void*>(cache));
  c.sb = strides[0];
  c.so = strides[1];
  c.sh = strides[2];
  c.skv = strides[3];
  c.num_blocks = static_cast<int32_t>(num_blocks);
  c.block_size = static_cast<int32_t>(block_size);
  c.div_bs = FastDiv(static_cast<uint32_t>(block_size));
  c.slots32 = num_blocks * block_size < (int64_t{1} << 31);
  c.heads = static_cast<int32_t>(heads);
  c.d = static_cast<int32_t>(d);
  c.W = static_cast<int32_t>(d / 8);
  c.NG = static_cast<int32_t>(fp4_groups(d));
  return EVS_OK;
}

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float scale_of(uint32_t byte) {
  return __builtin_bit_cast(float, byte << 23);  // 255 gives an exponent that converts to NaN
}

// Codes 2p and 2p + 1 of a dword, times the scale, as two bf16 in a dword.
template <int P>
__device__ __forceinline__ uint32_t codes_bf16(uint32_t dword, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(dword, scale, P));
}

// A dword's eight codes as the eight bf16 of an MFMA operand.
__device__ __forceinline__ bf16x8 codes8_bf16(uint32_t dword, float scale) {
  u32x4 r;
  r[0] = codes_bf16<0>(dword, scale);
  r[1] = codes_bf16<1>(dword, scale);
  r[2] = codes_bf16<2>(dword, scale);
  r[3] = codes_bf16<3>(dword, scale);
  return __builtin_bit_cast(bf16x8, r);
}

}  // namespace evs
