// Attention over a paged cache at full width (bf16 or f16), whose sequences may share prefixes: what
// its kernels share.
//
// The context of a query row (a query token and one of the heads that share a KV head) is its
// group's prefix and then its sequence's own tokens up to the query's. With s_t the scaled product
// of the query with token t's key,
//
//   out = sum_t exp(s_t - m) V_t / sum_t exp(s_t - m),   m = max_t s_t,   lse = m + ln(sum)
//
// and the sums over disjoint parts of the context join by their maxima: with (m_i, l_i, o_i) of part
// i and m = max m_i, l = sum l_i exp(m_i - m) and likewise o. So a prefix is taken once for the rows
// of all sequences of its group, and long contexts by several workgroups at once.
//
// Both products are MFMA tiles with f32 sums, computed transposed so that no value changes lanes
// between them: the scores leave a lane with four tokens of one query row, and those weights are its
// part of the second operand as they stand. A weight exp(s - m) is rounded to the cache's type before
// it multiplies V (bf16: at most 2^-8 of it, f16: 2^-11 or, below 2^-14, 2^-25 in all); the sum of
// the weights is taken before that. The matrix instructions take 16 bits, and a weight's rest as a
// second term would make them half as many again, which bound chunks, for less than the output's own
// rounding: answers are off from 64 bits by 0.0019 to 0.0023 of their norm in bf16 (f16: 0.00027),
// f32 sums rounded once by 0.0016 to 0.0017 (0.00021).
#pragma once

#include <type_traits>

#include "softmax.hpp"

namespace evs {

constexpr int kFullWaves = 4;
constexpr int kFullThreads = 64 * kFullWaves;
constexpr int kRowTile = 16;  // query rows that an MFMA tile has
// Sequences of up to kRowTile query rows a KV head take their own tokens in full_rows.hpp, others in
// full_tiles.hpp; those of up to kTogether take a prefix with the rest of their group, and longer
// chunks, which fill tiles by themselves, take it ahead of their own tokens, as one context.
// us where rows beyond 16, 64 and 256 do so, behind a prefix of 4 Ki: 8 chunks of 64 rows 53, 46 and
// 46; 8 of 128 rows 56, 56 and 53; 8 of 256 rows 87, 87 and 84; 64 of 128 rows 209, 206 and 249.
constexpr int kTogether = 64;
constexpr int kFullMinDim = 16;
constexpr int kFullMaxDim = 256;

// Contexts of one kind, in block tables.
struct Contexts {
  const int32_t* tables;
  int64_t stride;
  const int32_t* lens;
  int32_t width, n;
};

// How contexts are cut into parts, one a workgroup.
struct Cut {
  int32_t chunk, splits;  // a part's tokens, and the most parts of a context
  uint32_t tiles;         // row tiles that there may be
};

struct FullArgs {
  char* base;
  int64_t sb, so, sh, skv;  // page, slot in page, head, K to V, in bytes
  int32_t num_blocks, block_size;
  FastDiv div_bs;
  int32_t heads, d;
  const char* q;
  int64_t q_token, q_head;  // strides in bytes
  char* out;                // contiguous [tokens, q_heads, d]
  float* lse;               // contiguous [tokens, q_heads], or null
  float* top;               // the same in powers of two, for the weights, or null
  const int32_t* starts;    // null: one query a sequence
  int32_t seqs, tokens, max_q, q_heads;
  FastDiv shared, div_heads;
  float scale_log2;  // scale * log2(e)
  Contexts own, pre;
  const int32_t* group_starts;  // of the sequences of each prefix
  // how prefixes are cut for their groups' rows, own tokens for few rows, and contexts for many
  Cut group, few, many;
  bool few_groups;  // a group has at most kRowTile rows
  // Parts: sums [slots, rows, d], maxima and totals [slots, rows, 2]. `parts`: a row is a query and
  // head, and a slot a part of its group's prefix or, behind those, of a context for many rows.
  // `few_parts`: the slots are parts of own tokens for few rows, [seqs, heads, few_rows].
  struct Parts {
    float* sums;
    float* stats;
  } parts, few_parts;
  int32_t few_rows;
  int32_t row_tiles;  // of 16 rows, that a wave has of a tile of many
  // scores of few rows with their own tokens, for the weights: [seqs, heads, few_rows, stored], of
  // the first `stored` tokens; or null
  float* scores;
  int32_t stored;
  float* mass;  // [num_blocks, heads, block_size], or null
};

// Rows of queries and a context.
struct Rows {
  int32_t q0, nq;  // query tokens
  int32_t rows;    // query rows of a KV head
  int32_t len;     // tokens of the context
};

__device__ __forceinline__ int32_t length_of(const FullArgs& a, const Contexts& c, int i) {
  const int64_t room = static_cast<int64_t>(c.width) * a.block_size;
  const int32_t len = max(c.lens[i], 0);
  return a.num_blocks == 0 ? 0 : len > room ? static_cast<int32_t>(room) : len;
}

// Sequence s and its own tokens, kept within the arguments' bounds.
__device__ __forceinline__ Rows sequence_rows(const FullArgs& a, int s) {
  Rows r;
  if (a.starts == nullptr) {
    r.q0 = s;
    r.nq = 1;
  } else {
    r.q0 = max(a.starts[s], 0);
    r.nq = min(a.starts[s + 1], a.tokens) - r.q0;
    r.nq = max(min(r.nq, a.max_q), 0);
  }
  r.rows = r.nq * static_cast<int32_t>(a.shared.d);
  r.len = length_of(a, a.own, s);
  return r;
}

// The queries of group g's sequences, and its prefix.
__device__ __forceinline__ Rows group_rows(const FullArgs& a, int g) {
  const int s0 = min(max(a.group_starts[g], 0), a.seqs);
  const int s1 = min(max(a.group_starts[g + 1], s0), a.seqs);
  Rows r;
  r.q0 = a.starts == nullptr ? s0 : min(max(a.starts[s0], 0), a.tokens);
  const int end = a.starts == nullptr ? s1 : min(a.starts[s1], a.tokens);
  r.nq = max(end - r.q0, 0);
  r.rows = r.nq * static_cast<int32_t>(a.shared.d);
  r.len = length_of(a, a.pre, g);
  return r;
}

__device__ __forceinline__ Rows scalar_rows(Rows r) {
  r.q0 = __builtin_amdgcn_readfirstlane(r.q0);
  r.nq = __builtin_amdgcn_readfirstlane(r.nq);
  r.rows = __builtin_amdgcn_readfirstlane(r.rows);
  r.len = __builtin_amdgcn_readfirstlane(r.len);
  return r;
}

// Parts of the first `end` tokens of a context; the last that there may be takes the rest.
__device__ __forceinline__ int32_t parts_of(const Cut& c, int32_t end) {
  return end <= 0 ? 0 : min((end - 1) / c.chunk + 1, c.splits);
}

// Whether rows of a sequence with `rows` of them, whose own part of the context ends at `end`, are
// joined from parts. Of one part, without a prefix that others share, they are written where they go.
__device__ __forceinline__ bool is_joined(const FullArgs& a, const Cut& c, int32_t rows,
                                          int32_t end) {
  return parts_of(c, end) > 1 || (rows <= kTogether && a.group.tiles > 0);
}

// The one of `n` with place `at` on a line on which the rows rows_of(i) have count(rows) places, found
// by each wave for itself, without a wait for others; false past the line's end.
template <typename RowsOf, typename Count>
__device__ __forceinline__ bool find_rows(uint32_t n, uint32_t at, RowsOf rows_of, Count count,
                                          uint32_t& who, uint32_t& place, Rows& found) {
  const uint32_t lane = threadIdx.x & 63;
  for (uint32_t i0 = 0; i0 < n; i0 += 64) {
    Rows r{};
    if (i0 + lane < n) r = rows_of(i0 + lane);
    const uint32_t mine = i0 + lane < n ? count(r) : 0;
    uint32_t sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t up = __shfl_up(sum, d);
      if (lane >= static_cast<uint32_t>(d)) sum += up;
    }
    const unsigned long long hit = __builtin_amdgcn_ballot_w64(at < sum);
    if (hit != 0) {
      const int l = __builtin_ctzll(hit);
      who = i0 + l;
      place = at - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(mine, l));
      found.q0 = __builtin_amdgcn_readlane(r.q0, l);
      found.nq = __builtin_amdgcn_readlane(r.nq, l);
      found.rows = __builtin_amdgcn_readlane(r.rows, l);
      found.len = __builtin_amdgcn_readlane(r.len, l);
      return true;
    }
    at -= __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

// The last of the ascending at[0], ..., at[n - 1] that is at most x, by a wave; -1 if there is none.
__device__ __forceinline__ int last_at_most(const int32_t* at, int n, int x) {
  const int lane = threadIdx.x & 63;
  int lo = 0, span = n;
  while (span > 0) {
    const int step = (span + 63) >> 6;
    const int i = lane * step;
    const bool below = i < span && at[lo + i] <= x;
    const int k = __popcll(__builtin_amdgcn_ballot_w64(below));
    if (k == 0) return lo - 1;
    lo += (k - 1) * step;
    span -= (k - 1) * step;
    span = span < step ? span : step;
    if (span == 1) return lo;
  }
  return -1;
}

// The sequence that names query `token`, by a wave; -1 if none does.
__device__ __forceinline__ int sequence_of(const FullArgs& a, int token) {
  if (a.starts == nullptr) return token < a.seqs ? token : -1;
  const int s = __builtin_amdgcn_readfirstlane(last_at_most(a.starts, a.seqs, token));
  if (s < 0) return -1;
  const Rows r = scalar_rows(sequence_rows(a, s));
  return token >= r.q0 && token - r.q0 < r.nq ? s : -1;
}

// The group of sequence s, by a wave; -1 if it has no prefix.
__device__ __forceinline__ int group_of(const FullArgs& a, int s) {
  if (a.pre.n == 0) return -1;
  const int g = __builtin_amdgcn_readfirstlane(last_at_most(a.group_starts, a.pre.n, s));
  return g >= 0 && s < a.group_starts[g + 1] ? g : -1;
}

// ---------------------------------------------------------------- products
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// D[16, 16] += A[16, 32] B[32, 16]: lane l has eight elements of A's row l % 16 and of B's column
// l % 16, from 8 (l / 16) on, and of D's column l % 16 the rows 4 (l / 16) to + 3.
template <typename T>
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (std::is_same<T, __bf16>::value)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __bf16>::value) {
    return pack_bf16(lo, hi);
  } else {
    f16x2 v;
    v[0] = static_cast<_Float16>(lo);
    v[1] = static_cast<_Float16>(hi);
    return __builtin_bit_cast(uint32_t, v);
  }
}

// The bits of a half-word that are all set in an infinity and a NaN.
template <typename T>
constexpr uint32_t kWildBits = std::is_same<T, __bf16>::value ? 0x7F80u : 0x7C00u;

// A dword's two values without those that are no finite numbers.
template <typename T>
__device__ __forceinline__ uint32_t tamed(uint32_t x) {
  constexpr uint32_t lo = kWildBits<T>, hi = kWildBits<T> << 16;
  x = (x & lo) == lo ? x & 0xFFFF0000u : x;
  return (x & hi) == hi ? x & 0xFFFFu : x;
}
template <typename T>
__device__ __forceinline__ bool is_wild(uint32_t x) {
  constexpr uint32_t lo = kWildBits<T>, hi = kWildBits<T> << 16;
  return (x & lo) == lo || (x & hi) == hi;
}

// 16 bytes of a row that starts on 16.
__device__ __forceinline__ u32x4 load16(uint64_t p) {
  return *reinterpret_cast<const __attribute__((address_space(1))) u32x4*>(p);
}
__device__ __forceinline__ u32x2 load8(uint64_t p) {
  return *reinterpret_cast<const __attribute__((address_space(1))) u32x2*>(p);
}

// A query row's chunks of eight elements 4 i + quad, as operands; zeros past its end.
template <int NG>
__device__ __forceinline__ void load_query(const FullArgs& a, const char* p, int quad,
                                           u32x4 (&q)[NG]) {
#pragma unroll
  for (int i = 0; i < NG; i++) {
    const int c = 4 * i + quad;
    const bool in = 8 * c < a.d;
    const u32x4 x = load16(reinterpret_cast<uint64_t>(p) + (in ? 16 * c : 0));
#pragma unroll
    for (int k = 0; k < 4; k++) q[i][k] = in ? x[k] : 0;
  }
}

// Eight scores of this lane's row to weights, as an operand.
template <typename T>
__device__ __forceinline__ u32x4 full_weights(const float* s, float scale_log2, Running& r) {
  const float shift = r.shift();
  u32x4 p;
#pragma unroll
  for (int k = 0; k < 8; k += 2) {
    const float lo = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k], scale_log2, -shift));
    const float hi = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k + 1], scale_log2, -shift));
    r.l += lo + hi;
    p[k / 2] = pack2<T>(lo, hi);
  }
  return p;
}

// ---------------------------------------------------------------- results
// Where a part's row lies.
__device__ __forceinline__ int64_t part_at(const FullArgs& a, int32_t slot, int32_t token,
                                           int32_t q_head) {
  return (static_cast<int64_t>(slot) * a.tokens + token) * a.q_heads + q_head;
}
__device__ __forceinline__ int64_t few_part_at(const FullArgs& a, int32_t slot, int32_t seq,
                                               int32_t head, int32_t row) {
  return ((static_cast<int64_t>(slot) * a.seqs + seq) * a.heads + head) * a.few_rows + row;
}

__device__ __forceinline__ void keep4(const FullArgs::Parts& p, int d, int64_t at, int w, f32x4 v,
                                      float top, float total) {
  *reinterpret_cast<f32x4*>(p.sums + at * d + 4 * w) = v;
  if (w == 0) {
    p.stats[2 * at] = top;
    p.stats[2 * at + 1] = total;
  }
}

// Four elements of an output row, 4 w on, from the sums, their reference and the weights' total.
template <typename T>
__device__ __forceinline__ void finish4(const FullArgs& a, int32_t token, int32_t q_head, int w,
                                        f32x4 v, float top, float total) {
  const float inv = total > 0 ? 1.0f / total : (total == 0 ? 0.0f : total);  // NaN stays
  const int64_t at = static_cast<int64_t>(token) * a.q_heads + q_head;
  u32x2 y;
  y[0] = pack2<T>(v[0] * inv, v[1] * inv);
  y[1] = pack2<T>(v[2] * inv, v[3] * inv);
  *reinterpret_cast<u32x2*>(a.out + (at * a.d + 4 * w) * 2) = y;
  if (w == 0) {
    const float log2 = total == 0 ? -INFINITY : top + __builtin_amdgcn_logf(total);
    if (a.lse != nullptr) a.lse[at] = log2 * kLn2;
    // a row that sees nothing gives nothing
    if (a.top != nullptr) a.top[at] = total == 0 ? INFINITY : log2;
  }
}

// The products of the values that are no finite numbers among 32 tokens, whose rows are at `at` and
// whose scores for this lane's row are `s`: the row's elements get them if it sees the token, of
// which it sees those up to `ahead`. Such values are kept out of the other products, where a row
// ahead of the token would take them times 0.
template <typename T, int VW, int VD>
__device__ __forceinline__ void add_wild(const FullArgs& a, const uint64_t* at, uint32_t there,
                                         int ahead, const float* s, const Running& run,
                                         f32x4 (&o)[VD][VW]) {
  const int lane = lane_now();
  const int col = lane & 15, quad = lane >> 4;
  Running now = run;  // its shift is not to be shared with the weights', on the way of all tokens
  asm volatile("" : "+v"(now.m));
  const float shift = now.shift();
#pragma unroll 1
  for (int k = 0; k < 32; k++) {
    // the token's score is with the lanes of quarter k / 4 % 4
    float mine = s[0];
#pragma unroll
    for (int i = 1; i < 8; i++) mine = 4 * (k >> 4) + (k & 3) == i ? s[i] : mine;
    mine = __shfl(mine, col + 16 * ((k >> 2) & 3));
    if (!((there >> k) & 1) || k > ahead) continue;
    const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(mine, a.scale_log2, -shift));
    const uint64_t row = at[k] + a.skv;
#pragma unroll
    for (int v = 0; v < VD; v++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const uint64_t p = row + 2 * min(128 * v + VW * (4 * quad + r), a.d - VW);
        uint32_t x[VW / 2];
        if constexpr (VW == 8) {
          const u32x4 y = load16(p);
#pragma unroll
          for (int j = 0; j < 4; j++) x[j] = y[j];
        } else {
          const u32x2 y = load8(p);
          x[0] = y[0];
          x[1] = y[1];
        }
#pragma unroll
        for (int j = 0; j < VW; j++) {
          const uint16_t bits = static_cast<uint16_t>(x[j / 2] >> (16 * (j & 1)));
          const float y = w * static_cast<float>(__builtin_bit_cast(T, bits));
          o[v][j][r] += (bits & kWildBits<T>) == kWildBits<T> ? y : 0.0f;
        }
        __builtin_amdgcn_sched_barrier(0);  // few loads at once: registers are short
      }
  }
}

int full_attend(const FullArgs& a, int type, hipStream_t s);
int full_weigh(const FullArgs& a, int type, int64_t max_len, int64_t max_prefix, hipStream_t s);

}  // namespace evs
