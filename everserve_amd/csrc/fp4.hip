// Full-width K and V rows to 4-bit half-rows of a paged cache, and back (fp4.hpp has the format).
#include "fp4.hpp"

namespace evs {
namespace {

constexpr int kThreads = 256;

struct RowsIo {
  Fp4Cache c;
  const char* in[2];    // K and V rows (write)
  int64_t in_token[2];  // strides in bytes
  int64_t in_head[2];
  char* out[2];  // K and V rows, contiguous [n, heads, d] (read)
  const int64_t* slots;
  int64_t n;
  uint32_t units;     // work items of this launch
  FastDiv per_token;  // items a token has
  FastDiv per_half;   // items a head's row has
  bool vector;  // rows may be read in 16-byte words
};

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  return static_cast<float>(v);
}

// The half-row of slot `s`, head `h`; null for a slot the cache does not have (padding).
__device__ __forceinline__ char* half_row(const Fp4Cache& c, int64_t s, int h, int kv) {
  if (s < 0 || s >= static_cast<int64_t>(c.num_blocks) * c.block_size) return nullptr;
  int64_t block;
  if (c.slots32)
    block = c.div_bs.div(static_cast<uint32_t>(s));
  else
    block = s / c.block_size;
  const int64_t off = s - block * c.block_size;
  return c.base + block * c.sb + off * c.so + h * c.sh + kv * c.skv;
}

// Eight elements of a row as f32.
template <typename T>
__device__ __forceinline__ void load8(const char* p, bool vector, float (&x)[8]) {
  T v[8];
  if (vector) {
    __builtin_memcpy(v, __builtin_assume_aligned(p, 16), sizeof(v));
  } else {
    const T* e = reinterpret_cast<const T*>(p);
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = e[j];
  }
#pragma unroll
  for (int j = 0; j < 8; j++) x[j] = to_f32(v[j]);
}

__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  // lanes xor 1, then xor 2, of each four
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xB1, 0xF, 0xF, true)));
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x4E, 0xF, 0xF, true)));
  return v;
}

// Four lanes round a group of 32 elements, eight each. The scale is the least power of two, from
// 2^-126 to 2^125, that brings the group's largest magnitude to 7 or below: codes end at 6, the
// next would be 8, so up to 7 the largest element is off by no more than half a step, as the
// others are. (2^126 is left out because 4 times it is no finite bf16.) Codes are rounded to the
// nearest, ties to even, by the hardware's conversion.
//
// K's group and V's at the same place are one work item: they share the index arithmetic, and both
// their loads are under way before the first is needed (a call of 8,192 rows written and one of
// 32,768 read, 8 heads of 128: 50.8 us together, as two items 66.9).
//
// Bound by memory where there are many rows: 8,192 tokens of 8 heads of 128 in 11.0 us, 3.9 TB/s
// (a large plain copy reaches 4.84). A step's 64 rows are the launch alone (3.2 us).
template <typename T>
__global__ __launch_bounds__(kThreads) void write_rows(RowsIo a) {
  const uint32_t u = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t unit = u >> 2, lane = u & 3;
  if (unit >= a.units) return;  // whole groups of four lanes leave
  uint32_t token, rest, h, g;
  a.per_token.divmod(unit, token, rest);
  a.per_half.divmod(rest, h, g);
  const int64_t slot = a.slots[token];
  const uint32_t w = 4 * g + lane;  // this lane's dword of codes
  const bool in = w < static_cast<uint32_t>(a.c.W);
  float x[2][8] = {};
  if (in) {
#pragma unroll
    for (int kv = 0; kv < 2; kv++)
      load8<T>(a.in[kv] + token * a.in_token[kv] + h * a.in_head[kv] + w * (8 * sizeof(T)),
               a.vector, x[kv]);
  }
  char* row = half_row(a.c, slot, h, 0);
#pragma unroll
  for (int kv = 0; kv < 2; kv++) {
    // magnitudes compare as their bits do, an infinity and a NaN above every number
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 8; j++)
      most = max(most, __builtin_bit_cast(uint32_t, x[kv][j]) & 0x7FFFFFFFu);
    most = quad_max(most);
    const bool number = most < 0x7F800000u;
    // the exponent, and one more where the mantissa is above 1.75: 7 = 1.75 * 4
    const int e = static_cast<int>((most + 0x1FFFFFu) >> 23) - 2;
    const uint32_t byte = number ? static_cast<uint32_t>(min(max(e, 1), 252)) : kScaleNaN;
    uint32_t codes = 0;
    if (number) {
      const float s = scale_of(byte);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[kv][0], x[kv][1], s, 0);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[kv][2], x[kv][3], s, 1);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[kv][4], x[kv][5], s, 2);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[kv][6], x[kv][7], s, 3);
    }
    if (row == nullptr) continue;
    char* half = row + kv * a.c.skv;
    if (in) reinterpret_cast<uint32_t*>(half)[w] = codes;
    uint8_t* scales = reinterpret_cast<uint8_t*>(half + 4 * a.c.W);
    if (lane == 0) scales[g] = static_cast<uint8_t>(byte);
    // zeros after the last scale, up to a multiple of four bytes
    const uint32_t tail = a.c.NG & 3;
    if (lane > 0 && g == static_cast<uint32_t>(a.c.NG) - 1 && tail != 0 && lane <= 4 - tail)
      scales[a.c.NG + lane - 1] = 0;
  }
}

template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  return static_cast<T>(v);
}

// One lane turns a dword of K's codes and the one of V's at the same place into eight elements
// each, so that a wave's stores are whole lines. Bound by them: 32,768 tokens of 8 heads of 128 in
// bf16 in 32 us, 5.3 TB/s.
template <typename T>
__global__ __launch_bounds__(kThreads) void read_rows(RowsIo a) {
  const uint32_t unit = blockIdx.x * kThreads + threadIdx.x;
  if (unit >= a.units) return;
  uint32_t token, rest, h, w;
  a.per_token.divmod(unit, token, rest);
  a.per_half.divmod(rest, h, w);
  const char* row = half_row(a.c, a.slots[token], h, 0);
  uint32_t codes[2] = {0, 0};
  float s[2] = {1.0f, 1.0f};
  if (row != nullptr) {
#pragma unroll
    for (int kv = 0; kv < 2; kv++) {
      const char* half = row + kv * a.c.skv;
      codes[kv] = reinterpret_cast<const uint32_t*>(half)[w];
      s[kv] = scale_of(reinterpret_cast<const uint8_t*>(half)[4 * a.c.W + (w >> 2)]);
    }
  }
#pragma unroll
  for (int kv = 0; kv < 2; kv++) {
    const f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[kv], s[kv], 0);
    const f32x2 p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[kv], s[kv], 1);
    const f32x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[kv], s[kv], 2);
    const f32x2 p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[kv], s[kv], 3);
    T v[8];
    v[0] = from_f32<T>(p0[0]);
    v[1] = from_f32<T>(p0[1]);
    v[2] = from_f32<T>(p1[0]);
    v[3] = from_f32<T>(p1[1]);
    v[4] = from_f32<T>(p2[0]);
    v[5] = from_f32<T>(p2[1]);
    v[6] = from_f32<T>(p3[0]);
    v[7] = from_f32<T>(p3[1]);
    char* out = a.out[kv] + static_cast<int64_t>(unit) * static_cast<int64_t>(8 * sizeof(T));
    __builtin_memcpy(__builtin_assume_aligned(out, 16), v, sizeof(v));
  }
}

// Work items are counted in 32 bits: a longer list goes in several launches.
constexpr int64_t kMaxUnits = int64_t{1} << 28;

template <typename F>
int in_launches(RowsIo a, int64_t per_token, int lanes, const F& launch) {
  const int64_t most = kMaxUnits / per_token;
  for (int64_t t = 0; t < a.n; t += most) {
    RowsIo b = a;
    b.n = a.n - t < most ? a.n - t : most;
    b.units = static_cast<uint32_t>(b.n * per_token);
    b.slots = a.slots + t;
    for (int kv = 0; kv < 2; kv++) {
      if (a.in[kv] != nullptr) b.in[kv] = a.in[kv] + t * a.in_token[kv];
      if (a.out[kv] != nullptr) b.out[kv] = a.out[kv] + t * a.in_token[kv];
    }
    const uint32_t grid =
        static_cast<uint32_t>((static_cast<int64_t>(b.units) * lanes + kThreads - 1) / kThreads);
    launch(b, grid);
    EVS_LAUNCHED("fp4 rows");
  }
  return EVS_OK;
}

bool known_type(int type) { return type == EVS_BF16 || type == EVS_F16 || type == EVS_F32; }

}  // namespace
}  // namespace evs

extern "C" int evs_fp4_row_bytes(int64_t head_dim, int64_t* bytes) {
  evs::clear_error();
  EVS_REQUIRE(bytes != nullptr, "evs_fp4_row_bytes: null result");
  EVS_REQUIRE(head_dim >= evs::kFp4MinDim && head_dim <= evs::kFp4MaxDim && head_dim % 8 == 0,
              "evs_fp4_row_bytes: head size %lld: a multiple of 8 from %d to %d",
              static_cast<long long>(head_dim), evs::kFp4MinDim, evs::kFp4MaxDim);
  *bytes = evs::fp4_row_bytes(head_dim);
  return EVS_OK;
}

extern "C" int evs_fp4_write_rows(const void* key, const void* value, const int64_t* in_strides,
                                  int type, const int64_t* slots, int64_t n, void* cache,
                                  int64_t num_blocks, int64_t block_size, int64_t heads,
                                  int64_t head_dim, const int64_t* strides, void* stream) {
  evs::clear_error();
  const char* who = "evs_fp4_write_rows";
  EVS_REQUIRE(n >= 0, "%s: negative row count", who);
  EVS_REQUIRE(evs::known_type(type), "%s: element type %d", who, type);
  evs::RowsIo a{};
  if (const int rc =
          evs::fp4_cache(who, cache, num_blocks, block_size, heads, head_dim, strides, a.c))
    return rc;
  if (n == 0 || num_blocks == 0) return EVS_OK;
  EVS_REQUIRE(key != nullptr && value != nullptr && slots != nullptr && in_strides != nullptr,
              "%s: null rows, strides or slots", who);
  const int64_t elem = evs::elem_bytes(type);
  a.vector = true;
  const void* in[2] = {key, value};
  for (int kv = 0; kv < 2; kv++) {
    a.in[kv] = static_cast<const char*>(in[kv]);
    a.in_token[kv] = in_strides[2 * kv] * elem;
    a.in_head[kv] = in_strides[2 * kv + 1] * elem;
    EVS_REQUIRE(reinterpret_cast<uintptr_t>(in[kv]) % elem == 0, "%s: rows off their element size",
                who);
    a.vector = a.vector && reinterpret_cast<uintptr_t>(in[kv]) % 16 == 0 &&
               a.in_token[kv] % 16 == 0 && a.in_head[kv] % 16 == 0;
  }
  a.slots = slots;
  a.n = n;
  const int64_t per_token = heads * a.c.NG;
  a.per_token = evs::FastDiv(static_cast<uint32_t>(per_token));
  a.per_half = evs::FastDiv(static_cast<uint32_t>(a.c.NG));
  const hipStream_t s = evs::as_stream(stream);
  return evs::in_launches(a, per_token, 4, [&](const evs::RowsIo& b, uint32_t grid) {
    if (type == EVS_BF16)
      evs::write_rows<__bf16><<<grid, evs::kThreads, 0, s>>>(b);
    else if (type == EVS_F16)
      evs::write_rows<_Float16><<<grid, evs::kThreads, 0, s>>>(b);
    else
      evs::write_rows<float><<<grid, evs::kThreads, 0, s>>>(b);
  });
}

extern "C" int evs_fp4_read_rows(const void* cache, int64_t num_blocks, int64_t block_size,
                                 int64_t heads, int64_t head_dim, const int64_t* strides,
                                 const int64_t* slots, int64_t n, void* key, void* value, int type,
                                 void* stream) {
  evs::clear_error();
  const char* who = "evs_fp4_read_rows";
  EVS_REQUIRE(n >= 0, "%s: negative row count", who);
  EVS_REQUIRE(evs::known_type(type), "%s: element type %d", who, type);
  evs::RowsIo a{};
  if (const int rc =
          evs::fp4_cache(who, cache, num_blocks, block_size, heads, head_dim, strides, a.c))
    return rc;
  if (n == 0) return EVS_OK;
  EVS_REQUIRE(key != nullptr && value != nullptr && slots != nullptr, "%s: null rows or slots",
              who);
  EVS_REQUIRE((reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value)) % 16 == 0,
              "%s: the rows read must start on 16 bytes", who);
  a.out[0] = static_cast<char*>(key);
  a.out[1] = static_cast<char*>(value);
  a.in_token[0] = a.in_token[1] = heads * head_dim * evs::elem_bytes(type);
  a.slots = slots;
  a.n = n;
  const int64_t per_token = heads * a.c.W;
  a.per_token = evs::FastDiv(static_cast<uint32_t>(per_token));
  a.per_half = evs::FastDiv(static_cast<uint32_t>(a.c.W));
  const hipStream_t s = evs::as_stream(stream);
  return evs::in_launches(a, per_token, 1, [&](const evs::RowsIo& b, uint32_t grid) {
    if (type == EVS_BF16)
      evs::read_rows<__bf16><<<grid, evs::kThreads, 0, s>>>(b);
    else if (type == EVS_F16)
      evs::read_rows<_Float16><<<grid, evs::kThreads, 0, s>>>(b);
    else
      evs::read_rows<float><<<grid, evs::kThreads, 0, s>>>(b);
  });
}
