// Attention over a paged cache held in 4 bits (fp4.hpp has the format).
//
// For query row r of a sequence (a query token and one of the heads that share the KV head), with
// s_t = scale * sum_j q_j K_tj over the context's tokens t up to the query's own,
//
//   out = sum_t exp(s_t - m) V_t / sum_t exp(s_t - m),   m = max_t s_t,   lse = m + ln(sum)
//
// in one pass over the tokens with the running maximum and sum (both f32). Products are MFMA tiles
// of bf16 with f32 sums: a code times its scale is exact in bf16, so the scores' products are exact
// for bf16 queries; f16 queries go in as the sum of two bf16 (11 bits of mantissa fit in 8 + 8).
// The weights exp(s - m) are rounded to bf16 for the second product (at most half a step, 2^-8 of a
// weight, of either sign); their sum is taken before that rounding.
//
// Both products are computed transposed, so that no value changes lanes between them:
// - S^T = K Q^T: a lane of the first operand holds 8 x NW consecutive elements of one token (whole
//   dwords of codes), and the result leaves it with four tokens of one query row;
// - O^T = V^T P^T: those weights are a lane's part of the second operand as they stand, and a lane
//   of the first operand holds one dword of codes (eight elements) of eight tokens: it makes the
//   operands of eight products, one for each element.
#include "fp4.hpp"

namespace evs {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kRows = 16;  // query rows of a tile
constexpr int kTile = 32;  // tokens a wave takes at once

struct AttendArgs {
  Fp4Cache c;
  const char* q;
  int64_t q_token, q_head;  // strides in bytes
  bool q_vector;            // query rows may be read in 16-byte words
  char* out;                // contiguous [tokens, q_heads, d]
  float* lse;               // contiguous [tokens, q_heads], or null
  const int32_t* tables;
  int64_t table_stride;
  int32_t width;
  const int32_t* lens;
  const int32_t* starts;  // null: one query a sequence
  int32_t seqs, tokens, max_q, q_heads;
  FastDiv shared;      // query heads that share a KV head
  FastDiv heads;
  FastDiv q_tiles;     // row tiles a sequence may have
  float scale_log2;    // scale * log2(e)
};

// What a sequence's work is, from the device's arrays, kept within the arguments' bounds.
struct Sequence {
  int32_t q0, nq;  // its queries
  int32_t len;     // its context
  int32_t rows;    // query rows of a KV head
};

__device__ __forceinline__ Sequence sequence(const AttendArgs& a, int s) {
  Sequence r;
  if (a.starts == nullptr) {
    r.q0 = s;
    r.nq = 1;
  } else {
    r.q0 = max(a.starts[s], 0);
    r.nq = min(a.starts[s + 1], a.tokens) - r.q0;
    r.nq = max(min(r.nq, a.max_q), 0);
  }
  const int64_t room = static_cast<int64_t>(a.width) * a.c.block_size;
  int32_t len = max(a.lens[s], 0);
  if (len > room) len = static_cast<int32_t>(room);
  r.len = a.c.num_blocks > 0 ? len : 0;
  r.rows = r.nq * static_cast<int32_t>(a.shared.d);
  return r;
}

template <typename T>
struct QueryTerms;  // bf16 terms a query is the sum of
template <>
struct QueryTerms<__bf16> {
  static constexpr int n = 1;
};
template <>
struct QueryTerms<_Float16> {
  static constexpr int n = 2;
};

// NW consecutive dwords at any multiple of 4 bytes.
template <int NW>
struct Dwords {
  uint32_t v[NW];
};

template <int NW>
__device__ __forceinline__ Dwords<NW> load_dwords(const char* p) {
  Dwords<NW> r;
  __builtin_memcpy(&r, __builtin_assume_aligned(p, 4), sizeof(r));
  return r;
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

// One workgroup: a tile of 16 query rows of one KV head of one sequence. Its waves take the
// context's tokens in turns, 32 at a time, and join their results in LDS.
template <int NW, int VD, typename T>
__global__ __launch_bounds__(kThreads) void attend_rows(AttendArgs a) {
  constexpr int kTerms = QueryTerms<T>::n;
  constexpr int kDims = 128 * VD;  // the output tile's width, its padding included
  __shared__ float s_o[kWaves][kRows][kDims + 4];
  __shared__ float s_m[kWaves][kRows];
  __shared__ float s_l[kWaves][kRows];

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 15, quad = lane >> 4;
  uint32_t seq, head, tile, rest;
  a.heads.divmod(blockIdx.x, rest, head);
  a.q_tiles.divmod(rest, seq, tile);
  const Sequence sq = sequence(a, seq);
  const int row0 = tile * kRows;
  if (row0 >= sq.rows) return;
  const int last_row = min(row0 + kRows, sq.rows) - 1;

  // this lane's query row, and the tokens that it sees: those up to `sees`
  const int row = min(row0 + col, last_row);
  uint32_t qi, qg;
  a.shared.divmod(row, qi, qg);
  const int sees = sq.len - sq.nq + static_cast<int>(qi);
  const int end = min(sq.len, sq.len - sq.nq + static_cast<int>(a.shared.div(last_row)) + 1);

  // The query operands. Quarter `quad` of the lanes holds the codes' dwords [quad * NW, +NW), moved
  // back where they would pass the half-row's end: the query is zero for those seen twice.
  const int W = a.c.W;
  const int w0 = min(quad * NW, W - NW);
  bf16x8 qf[kTerms][NW];
  {
    const char* qp = a.q + (sq.q0 + qi) * a.q_token + (head * a.shared.d + qg) * a.q_head;
#pragma unroll
    for (int i = 0; i < NW; i++) {
      T v[8];
      const char* p = qp + (w0 + i) * 16;
      if (a.q_vector) {
        __builtin_memcpy(v, __builtin_assume_aligned(p, 16), 16);
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = reinterpret_cast<const T*>(p)[j];
      }
      const bool own = w0 + i >= quad * NW;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float x = own ? static_cast<float>(v[j]) : 0.0f;
        const __bf16 hi = static_cast<__bf16>(x);
        qf[0][i][j] = hi;
        if (kTerms > 1) qf[kTerms - 1][i][j] = static_cast<__bf16>(x - static_cast<float>(hi));
      }
    }
  }

  const char* base = a.c.base + head * a.c.sh;
  const int32_t* table = a.tables + static_cast<int64_t>(seq) * a.table_stride;
  // the half-row K of token t; `ok`: t is in the context and its page in the cache
  const auto row_of = [&](int t, bool& ok) {
    uint32_t page, off;
    a.c.div_bs.divmod(min(t, end - 1), page, off);
    const int32_t block = table[page];
    ok = t < end && block >= 0 && block < a.c.num_blocks;
    return base + (ok ? block : 0) * a.c.sb + off * a.c.so;
  };

  f32x4 o[VD][8];
#pragma unroll
  for (int v = 0; v < VD; v++)
#pragma unroll
    for (int j = 0; j < 8; j++) o[v][j] = f32x4{0, 0, 0, 0};
  float m = -INFINITY, l = 0;  // this lane's row's running maximum (scaled), its part of the sum

  for (int t0 = wave * kTile; t0 < end; t0 += kWaves * kTile) {
    float s[8];
    bool ok[8];
    const char* vrow[8];
#pragma unroll
    for (int g = 0; g < 2; g++) {
      bool k_ok;
      const char* p = row_of(t0 + 16 * g + col, k_ok);
      const Dwords<NW> codes = load_dwords<NW>(p + 4 * w0);
      f32x4 acc = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < NW; i++) {
        const float sc =
            scale_of(reinterpret_cast<const uint8_t*>(p)[4 * W + ((w0 + i) >> 2)]);
        const bf16x8 k = codes8_bf16(codes.v[i], sc);
#pragma unroll
        for (int n = 0; n < kTerms; n++)
          acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, qf[n][i], acc, 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int t = t0 + 16 * g + 4 * quad + r;
        vrow[4 * g + r] = row_of(t, ok[4 * g + r]) + a.c.skv;
        s[4 * g + r] = ok[4 * g + r] && t <= sees ? acc[r] * a.scale_log2 : -INFINITY;
      }
    }
    float top = s[0];
#pragma unroll
    for (int k = 1; k < 8; k++) top = fmaxf(top, s[k]);
    top = fmaxf(across_rows_max(top), m);
    const float shift = top == -INFINITY ? 0.0f : top;  // a row that has seen nothing yet
    const float fade = __builtin_amdgcn_exp2f(m - shift);
    m = top;
    float sum = 0;
    u32x4 p;
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
      const float lo = __builtin_amdgcn_exp2f(s[k] - shift);
      const float hi = __builtin_amdgcn_exp2f(s[k + 1] - shift);
      sum += lo + hi;
      p[k / 2] = pack_bf16(lo, hi);
    }
    l = l * fade + sum;
    const bf16x8 pf = __builtin_bit_cast(bf16x8, p);
#pragma unroll
    for (int v = 0; v < VD; v++) {
      const int w = min(16 * v + col, W - 1);
      uint32_t code[8];
      float sc[8];
#pragma unroll
      for (int k = 0; k < 8; k++) {
        code[k] = load_dwords<1>(vrow[k] + 4 * w).v[0];
        // a token outside the context must be a number, whatever its row holds: its weight is 0
        sc[k] = ok[k] ? scale_of(reinterpret_cast<const uint8_t*>(vrow[k])[4 * W + (w >> 2)])
                      : 1.0f;
      }
      // elements 2c and 2c + 1 of the eight tokens
      const auto pair = [&](auto c_) {
        constexpr int c = decltype(c_)::value;
        u32x4 even, odd;
#pragma unroll
        for (int k = 0; k < 8; k += 2) {
          const uint32_t x = codes_bf16<c>(code[k], sc[k]);
          const uint32_t y = codes_bf16<c>(code[k + 1], sc[k + 1]);
          even[k / 2] = __builtin_amdgcn_perm(y, x, 0x05040100u);
          odd[k / 2] = __builtin_amdgcn_perm(y, x, 0x07060302u);
        }
        o[v][2 * c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, even), pf,
                                                              o[v][2 * c] * fade, 0, 0, 0);
        o[v][2 * c + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            __builtin_bit_cast(bf16x8, odd), pf, o[v][2 * c + 1] * fade, 0, 0, 0);
      };
      pair(std::integral_constant<int, 0>{});
      pair(std::integral_constant<int, 1>{});
      pair(std::integral_constant<int, 2>{});
      pair(std::integral_constant<int, 3>{});
    }
  }
  l = across_rows_sum(l);

  // Join the waves: element 8 (4 quad + r) + j of row `col` is o[v][j][r].
#pragma unroll
  for (int v = 0; v < VD; v++)
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
      for (int j = 0; j < 8; j++)
        s_o[wave][col][128 * v + 8 * (4 * quad + r) + j] = o[v][j][r];
  if (quad == 0) {
    s_m[wave][col] = m;
    s_l[wave][col] = l;
  }
  __syncthreads();
  for (int x = threadIdx.x; x < kRows * a.c.W; x += kThreads) {
    const int r = x / a.c.W, w = x - r * a.c.W;
    if (row0 + r > last_row) break;  // rows ascend
    float top = s_m[0][r];
#pragma unroll
    for (int k = 1; k < kWaves; k++) top = fmaxf(top, s_m[k][r]);
    const float shift = top == -INFINITY ? 0.0f : top;
    float total = 0, v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < kWaves; k++) {
      const float f = __builtin_amdgcn_exp2f(s_m[k][r] - shift);
      total += f * s_l[k][r];
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] += f * s_o[k][r][8 * w + j];
    }
    const float inv = total > 0 ? 1.0f / total : (total == 0 ? 0.0f : total);
    uint32_t i, g;
    a.shared.divmod(row0 + r, i, g);
    const int64_t at =
        static_cast<int64_t>(sq.q0 + i) * a.q_heads + head * a.shared.d + g;
    T y[8];
#pragma unroll
    for (int j = 0; j < 8; j++) y[j] = static_cast<T>(v[j] * inv);
    __builtin_memcpy(__builtin_assume_aligned(a.out + (at * a.c.W + w) * 16, 16), y, 16);
    if (w == 0 && a.lse != nullptr)
      a.lse[at] = total == 0 ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * 0.6931471805599453f;
  }
}

template <int NW, int VD>
int launch(const AttendArgs& a, int type, uint32_t grid, hipStream_t s) {
  if (type == EVS_BF16)
    attend_rows<NW, VD, __bf16><<<grid, kThreads, 0, s>>>(a);
  else
    attend_rows<NW, VD, _Float16><<<grid, kThreads, 0, s>>>(a);
  EVS_LAUNCHED("evs_fp4_attend");
  return EVS_OK;
}

}  // namespace
}  // namespace evs

extern "C" int evs_fp4_attend_workspace(int64_t seqs, int64_t tokens, int64_t q_heads,
                                        int64_t heads, int64_t head_dim, int64_t max_q,
                                        int64_t max_len, int64_t* bytes) {
  evs::clear_error();
  EVS_REQUIRE(bytes != nullptr, "evs_fp4_attend_workspace: null result");
  *bytes = 0;
  return EVS_OK;
}

extern "C" int evs_fp4_attend(const void* q, const int64_t* q_strides, int type, void* out,
                              float* lse, int64_t tokens, int64_t q_heads, const void* cache,
                              int64_t num_blocks, int64_t block_size, int64_t heads,
                              int64_t head_dim, const int64_t* strides, const int32_t* tables,
                              int64_t table_stride, int64_t width, const int32_t* lens,
                              const int32_t* q_starts, int64_t seqs, int64_t max_q,
                              int64_t max_len, float scale, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  evs::clear_error();
  const char* who = "evs_fp4_attend";
  EVS_REQUIRE(type == EVS_BF16 || type == EVS_F16, "%s: query type %d: bf16 or f16", who, type);
  evs::AttendArgs a{};
  if (const int rc =
          evs::fp4_cache(who, cache, num_blocks, block_size, heads, head_dim, strides, a.c))
    return rc;
  EVS_REQUIRE(tokens >= 0 && tokens < (int64_t{1} << 31) && seqs >= 0 &&
                  seqs < (int64_t{1} << 31) && max_q >= 0 && width >= 0 &&
                  width < (int64_t{1} << 31) && max_len >= 0,
              "%s: bad count", who);
  EVS_REQUIRE(q_heads > 0 && q_heads < (int64_t{1} << 16) && q_heads % heads == 0,
              "%s: %lld query heads on %lld", who, static_cast<long long>(q_heads),
              static_cast<long long>(heads));
  EVS_REQUIRE(scale > 0 && scale < INFINITY, "%s: the scale must be positive and finite", who);
  if (tokens == 0 || seqs == 0 || max_q == 0) return EVS_OK;
  EVS_REQUIRE(q_starts != nullptr || (tokens == seqs && max_q == 1),
              "%s: without query starts there is one query a sequence: %lld queries, %lld sequences",
              who, static_cast<long long>(tokens), static_cast<long long>(seqs));
  EVS_REQUIRE(q != nullptr && q_strides != nullptr && out != nullptr && lens != nullptr &&
                  (tables != nullptr || width == 0),
              "%s: null argument", who);
  EVS_REQUIRE(reinterpret_cast<uintptr_t>(out) % 16 == 0, "%s: out must start on 16 bytes", who);
  EVS_REQUIRE(reinterpret_cast<uintptr_t>(q) % 2 == 0, "%s: queries off their element size", who);
  a.q = static_cast<const char*>(q);
  a.q_token = q_strides[0] * 2;
  a.q_head = q_strides[1] * 2;
  a.q_vector = reinterpret_cast<uintptr_t>(q) % 16 == 0 && a.q_token % 16 == 0 &&
               a.q_head % 16 == 0;
  a.out = static_cast<char*>(out);
  a.lse = lse;
  a.tables = tables;
  a.table_stride = table_stride;
  a.width = static_cast<int32_t>(width);
  a.lens = lens;
  a.starts = q_starts;
  a.seqs = static_cast<int32_t>(seqs);
  a.tokens = static_cast<int32_t>(tokens);
  if (max_q > tokens) max_q = tokens;
  a.max_q = static_cast<int32_t>(max_q);
  a.q_heads = static_cast<int32_t>(q_heads);
  const int64_t shared = q_heads / heads;
  a.shared = evs::FastDiv(static_cast<uint32_t>(shared));
  a.heads = evs::FastDiv(static_cast<uint32_t>(heads));
  a.scale_log2 = scale * 1.4426950408889634f;
  EVS_REQUIRE(max_q * shared < (int64_t{1} << 31), "%s: too many query rows", who);
  const int64_t q_tiles = (max_q * shared + evs::kRows - 1) / evs::kRows;
  a.q_tiles = evs::FastDiv(static_cast<uint32_t>(q_tiles));
  EVS_REQUIRE(q_tiles * heads < (int64_t{1} << 31) &&
                  q_tiles * heads * seqs < (int64_t{1} << 24),
              "%s: %lld tiles of query rows: at most 2^24", who,
              static_cast<long long>(q_tiles * heads * seqs));
  const uint32_t grid = static_cast<uint32_t>(q_tiles * heads * seqs);
  const hipStream_t s = evs::as_stream(stream);
  const int64_t per = (a.c.W + 3) / 4;  // dwords of codes a quarter of the lanes holds
  if (per <= 2) return evs::launch<2, 1>(a, type, grid, s);
  if (per <= 3) return evs::launch<3, 1>(a, type, grid, s);
  if (per <= 4) return evs::launch<4, 1>(a, type, grid, s);
  if (per <= 6) return evs::launch<6, 2>(a, type, grid, s);
  return evs::launch<8, 2>(a, type, grid, s);
}
