// Attention over a paged cache held in 4 bits (fp4.hpp has the format): what its kernels share.
//
// For query row r of a sequence (a query token and one of the heads that share the KV head), with
// s_t = scale * sum_j q_j K_tj over the context's tokens t up to the query's own,
//
//   out = sum_t exp(s_t - m) V_t / sum_t exp(s_t - m),   m = max_t s_t,   lse = m + ln(sum)
//
// in one pass over the tokens with the running maximum and sum (both f32).
//
// Products are MFMA tiles of bf16 with f32 sums: a code times its scale is exact in bf16, so the
// scores' products are exact for bf16 queries; f16 queries go in as the sum of two bf16 (11 bits of
// mantissa fit in 8 + 8). The weights exp(s - m) are rounded to bf16 for bf16 outputs (at most half
// a step, 2^-8 of a weight, of either sign; their sum is taken before that) and are the sum of two
// bf16 for f16 ones (off by 2^-17). The scaled MFMA, which would take K's codes and scales as they
// lie in the cache, is not used for the scores: with queries as sums of e4m3 terms its sums were
// off by 2^-13 to 2^-17 of the products' magnitudes, where these are off by 2^-24.
//
// Both products are computed transposed, so that no value changes lanes between them: the scores
// leave a lane with four tokens of one query row, and those weights are its part of the second
// operand as they stand.
#pragma once

#include "fp4.hpp"

namespace evs {

constexpr int kFewWaves = 8;   // of a workgroup, at most
constexpr int kManyWaves = 4;
constexpr float kLn2 = 0.6931471805599453f;

// Sequences with at most `few_rows` query rows a KV head (the call chooses) go to attend_few in
// tiles of 16, others to attend_many in tiles of 128, of 64 for head sizes above 128 (their sums
// take twice the registers).
constexpr int kFewTile = 16;
constexpr int many_tile(int64_t head_dim) { return head_dim > 128 ? 64 : 128; }

// How one kernel's work is dealt out (see Share below and `deal`).
struct Dealt {
  uint32_t workgroups;  // a KV head (few: a group of them) has, a multiple of 8
  bool split;           // contexts may be split between workgroups
  uint32_t tile_bits;   // log2 of a tile's rows
  int32_t rows;         // of them that are ever used
  float* part;  // [workgroups, 2, heads, rows, d + 2]: a part's sums, running maximum and total
  // Which shares a split tile is in, for the join. few: [seqs, tiles a sequence may have], the
  // first and how many (tiles of 16 rows are many, but few of a sequence); many: [workgroups], of
  // the share with the tile's start, the sequence, the tile and how many, below 2 if there is none.
  uint4* tiles_in;
  int64_t in;    // entries of it
  FastDiv most;  // tiles that a sequence may have
};

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
  float scale_log2;    // scale * log2(e)
  FastDiv held;        // KV heads that a workgroup of attend_few takes
  uint32_t turns;      // and waves that each of them has
  FastDiv one;
  FastDiv groups;      // such groups of heads
  uint32_t join_bits;  // log2 of a joined row's dwords, rounded up
  FastDiv heads;
  int32_t few_rows;
  Dealt few, many;
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

// The sequence of a whole workgroup, in scalars.
__device__ __forceinline__ Sequence sequence_of_all(const AttendArgs& a, uint32_t s) {
  Sequence r = sequence(a, static_cast<int>(s));
  r.q0 = __builtin_amdgcn_readfirstlane(r.q0);
  r.nq = __builtin_amdgcn_readfirstlane(r.nq);
  r.len = __builtin_amdgcn_readfirstlane(r.len);
  r.rows = __builtin_amdgcn_readfirstlane(r.rows);
  return r;
}

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

// Row tiles of a sequence in the kernel for many rows, or in that for few.
template <bool kMany>
__device__ __forceinline__ uint32_t tiles_of(const AttendArgs& a, const Sequence& q) {
  const uint32_t bits = (kMany ? a.many : a.few).tile_bits;
  return (q.rows > a.few_rows) == kMany ? (q.rows + (1u << bits) - 1) >> bits : 0;
}

// Stages of `tokens` that a row tile takes; an empty context takes one too, that it is answered. On
// the line every tile of a sequence takes the whole context, though those ahead of the last see
// less of it: where most of a context is queries, shares are unlike. Of one prompt of 4,096 tokens
// the busiest share has 1.9 times the mean's work (449 TFLOP/s), of chunks behind a prefix of
// 3 to 7 Ki tokens 1.1 times (713).
__device__ __forceinline__ uint32_t stages_of(const Sequence& q, uint32_t tokens) {
  return q.len <= 0 ? 1 : (q.len + tokens - 1) / tokens;
}

// A workgroup's share of the work. All row tiles' stages, sequence by sequence and tile by tile,
// are one line, cut into equal shares: a workgroup may have the end of a tile, some whole tiles and
// the start of another. Each finds its share by itself from the lengths, so nothing is planned
// ahead of the launch. Without splits the line is of whole tiles, one a share.
//
// A tile costs its workgroup a start (its queries, its first pages and rows) beside its stages: on
// the line it has kStart places more, ahead of them.
//
// A tile in several shares is joined from their parts: the share with the tile's start keeps its
// part in slot 1, those after it in slot 0.
struct Share {
  uint32_t seq, tile, first;  // the first place of it
  uint32_t count;             // places
  unsigned long long line, size;  // the tile's start on the line, places of a share
};
template <bool kMany>
constexpr uint32_t kStart = kMany ? 2 : 3;  // a start took 2 to 4 times as long as a stage

// The fewest stages of a share, in tokens; contexts of up to twice as many are not split. With half
// as many a context of 600 tokens took 13.4 us for 12.3 and 16 sequences of up to 2,000 21.2 for
// 21.8. With twice as many one of 4,000 took 19.0 for 17.5, and a batch with one long chunk 107 for
// 99; 4 sequences of 4 to 8 Ki with 128 rows 80 for 100.
constexpr uint32_t kMinShare = 512;

// Without splits, in the kernel for many rows: row tile `at` from the sequence with the longest
// context on, and in a sequence from the last one on, which see the most tokens. Workgroups start
// in this order, so that the last to start have the least to do. For at most as many sequences as
// threads.
__device__ __forceinline__ bool longest_first(const AttendArgs& a, uint32_t at, Share& r) {
  __shared__ int32_t s_len[64 * kManyWaves];
  __shared__ uint32_t s_tiles[64 * kManyWaves];
  __shared__ uint32_t s_found[2];
  const int tid = threadIdx.x;
  Sequence q{};
  if (tid < a.seqs) q = sequence(a, tid);
  const uint32_t tiles = tid < a.seqs ? tiles_of<true>(a, q) : 0;
  s_len[tid] = q.len;
  s_tiles[tid] = tiles;
  if (tid == 0) s_found[0] = 0xFFFFFFFFu;
  __syncthreads();
  unsigned long long before = 0;
  for (int s = 0; s < a.seqs; s++)
    if (s_len[s] > q.len || (s_len[s] == q.len && s < tid)) before += s_tiles[s];
  if (at >= before && at - before < tiles) {
    s_found[0] = tid;
    s_found[1] = tiles - 1 - static_cast<uint32_t>(at - before);
  }
  __syncthreads();
  r.seq = __builtin_amdgcn_readfirstlane(s_found[0]);
  r.tile = __builtin_amdgcn_readfirstlane(s_found[1]);
  r.first = 0;
  r.count = 1;
  return r.seq != 0xFFFFFFFFu;
}

// Share `at` of the line. False: past its end.
template <bool kMany>
__device__ __forceinline__ bool find_share(const AttendArgs& a, uint32_t at, uint32_t tokens,
                                           Share& r) {
  typedef unsigned long long u64;
  __shared__ u64 s_wave[kFewWaves];
  __shared__ uint32_t s_seq, s_place;
  const Dealt& dealt = kMany ? a.many : a.few;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int threads = blockDim.x, waves = threads >> 6;
  const auto length = [&](int s) -> u64 {
    if (s >= a.seqs) return 0;
    const Sequence q = sequence(a, s);
    const uint32_t tiles = tiles_of<kMany>(a, q);
    return dealt.split ? static_cast<u64>(tiles) * (kStart<kMany> + stages_of(q, tokens)) : tiles;
  };
  // the line's length, and the places of the first sequences, which are often all of them
  u64 total = 0;
  u64 mine = length(tid);
  if (a.seqs > threads) {
    u64 rest = 0;
    for (int s = tid + threads; s < a.seqs; s += threads) rest += length(s);
    rest = wave_sum(rest);
    if (lane == 0) s_wave[wave] = rest;
    __syncthreads();
    for (int k = 0; k < waves; k++) total += s_wave[k];
  }
  if (tid == 0) s_seq = 0xFFFFFFFFu;
  u64 start = 0, before = 0;
  r.size = 1;
  for (int s0 = 0; s0 < a.seqs; s0 += threads) {
    if (s0 > 0) mine = length(s0 + tid);
    u64 sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const u64 up = __shfl_up(sum, d);
      if (lane >= d) sum += up;
    }
    __syncthreads();
    if (lane == 63) s_wave[wave] = sum;
    __syncthreads();
    u64 from = before + sum - mine;
    for (int k = 0; k < waves; k++) {
      if (k < wave) from += s_wave[k];
      before += s_wave[k];
    }
    if (s0 == 0) {
      total = scalar(total + before);
      if (dealt.split) {
        const u64 least = (kMinShare + tokens - 1) / tokens;
        r.size = (total + dealt.workgroups - 1) / dealt.workgroups;
        r.size = scalar(r.size < least ? least : r.size);
      }
      start = at * r.size;
      if (start >= total) return false;  // uniform
    }
    if (start >= from && start - from < mine) {
      s_seq = s0 + tid;
      s_place = static_cast<uint32_t>(start - from);
    }
    if (start < before) break;
  }
  __syncthreads();
  r.seq = __builtin_amdgcn_readfirstlane(s_seq);
  if (r.seq == 0xFFFFFFFFu) return false;
  const uint32_t place = __builtin_amdgcn_readfirstlane(s_place);
  const uint32_t places =
      dealt.split ? kStart<kMany> + stages_of(sequence_of_all(a, r.seq), tokens) : 1;
  r.tile = place / places;
  r.first = place - r.tile * places;
  r.line = scalar(start - r.first);
  const u64 left = total - start;
  r.count = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(left < r.size ? left : r.size));
  return true;
}

// The part of a share in one row tile.
struct Part {
  int32_t row0, last_row;  // rows of the sequence
  int32_t begin, stop;     // tokens, up to the last that some row sees
  bool none;               // no stage of it (the share ends ahead of the first)
  bool whole;              // all of the tile
  uint32_t places;         // of the tile
  uint32_t slot;           // of the parts, if not
};

// The share's next part; it is taken off the share, which is left at the tile's end.
template <bool kMany>
__device__ __forceinline__ Part next_part(const AttendArgs& a, const Sequence& sq, Share& r,
                                          uint32_t tokens) {
  const uint32_t bits = (kMany ? a.many : a.few).tile_bits;
  Part p;
  p.row0 = static_cast<int>(r.tile << bits);
  p.last_row = min(p.row0 + (1 << bits), sq.rows) - 1;
  const int end = min(sq.len, sq.len - sq.nq + static_cast<int>(a.shared.div(p.last_row)) + 1);
  const bool split = (kMany ? a.many : a.few).split;
  const uint32_t start = split ? kStart<kMany> : 0, stages = split ? stages_of(sq, tokens) : 1;
  const uint32_t take = min(start + stages - r.first, r.count);
  const uint32_t from = max(r.first, start) - start, to = max(r.first + take, start) - start;
  p.none = from == to;
  p.places = start + stages;
  p.whole = to - from == stages;
  p.slot = from == 0 ? 1 : 0;
  p.begin = static_cast<int>(from * tokens);
  p.stop = to == stages ? end : min(end, static_cast<int>(to * tokens));
  r.count -= take;
  return p;
}

// On to the next tile, of the next sequence that has one (there is one while the share's count is
// above zero).
template <bool kMany>
__device__ __forceinline__ void next_tile(const AttendArgs& a, const Part& p, Share& r,
                                          Sequence& sq) {
  r.first = 0;
  r.line += p.places;
  if (++r.tile < tiles_of<kMany>(a, sq)) return;
  r.tile = 0;
  while (static_cast<int>(++r.seq) < a.seqs) {
    sq = sequence_of_all(a, r.seq);
    if (tiles_of<kMany>(a, sq) > 0) return;
  }
  r.count = 0;
}

// The lane's number, afresh: what is computed from it is computed in every part, where the compiler
// would move it ahead of all parts and keep it in registers that the stages need.
__device__ __forceinline__ int lane_now() {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  return lane;
}

// The kernel's arguments, read afresh, for the same reason: what a part's start and end need of
// them is not to take the stages' scalar registers.
__device__ __forceinline__ AttendArgs args_now() {
  uint64_t p = reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr());
  asm volatile("" : "+s"(p));
  AttendArgs a;
  typedef const __attribute__((address_space(4))) char* Constant;
  __builtin_memcpy(&a, (const void*)reinterpret_cast<Constant>(p), sizeof(a));
  return a;
}

// bf16 terms that a query, and a weight for such a query's output, is the sum of.
template <typename T>
struct QueryTerms;
template <>
struct QueryTerms<__bf16> {
  static constexpr int n = 1;
};
template <>
struct QueryTerms<_Float16> {
  static constexpr int n = 2;
};

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

// ---------------------------------------------------------------- scores
// Which dword of a half-row's codes product i of the scores takes from quarter `quad` of the lanes:
// any order will do that is the same for K and the queries. Where the groups are a multiple of
// four, a quarter has a group's four dwords (one wide read, one scale) for four products; of two
// groups, half of one for two products; else product i is group i.
template <int NG>
struct Order {
  static constexpr int kRun = NG % 4 == 0 ? 4 : NG == 2 ? 2 : 1;  // dwords read at once
  static __device__ __forceinline__ int dword(int i, int quad) {
    return kRun == 1 ? 4 * i + quad : 16 * (i / 4) + kRun * quad + i % kRun;
  }
};

// A row's query as operands; elements past its end are zeros.
template <int NG, typename T>
struct Query {
  static constexpr int kTerms = QueryTerms<T>::n;
  bf16x8 terms[kTerms][NG];

  __device__ __forceinline__ void load(const AttendArgs& a, const char* qp, int quad) {
#pragma unroll
    for (int i = 0; i < NG; i++) {
      const int w = Order<NG>::dword(i, quad);
      const bool in = w < a.c.W;
      const char* p = qp + (in ? w : 0) * 16;
      T v[8];
      if (a.q_vector) {
        __builtin_memcpy(v, __builtin_assume_aligned(p, 16), 16);
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = reinterpret_cast<const T*>(p)[j];
      }
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float x = in ? static_cast<float>(v[j]) : 0.0f;
        const __bf16 hi = static_cast<__bf16>(x);
        terms[0][i][j] = hi;
        if (kTerms > 1) terms[kTerms - 1][i][j] = static_cast<__bf16>(x - static_cast<float>(hi));
      }
    }
  }
};

// Token t's place among the rows of its 16: a lane's four tokens lie four rows apart, so that the
// four quarters of a wave read different banks.
__device__ __forceinline__ uint32_t place_of(uint32_t t) {
  return (t & ~15u) | ((t & 3) << 2) | ((t >> 2) & 3);
}

// The scores of 32 tokens, whose codes and scales lie in LDS from row `at` on, with 16 rows'
// queries, kTiles times over.
template <int NG, int kTiles, typename T, typename Lds>
__device__ __forceinline__ void scores(const Lds& lds, int at, int lane, int W,
                                       const Query<NG, T> (&q)[kTiles], f32x4 (&acc)[2][kTiles]) {
  constexpr int kRun = Order<NG>::kRun;
  const int quad = lane >> 4, col = lane & 15;
  const int row = at + place_of(col);
#pragma unroll
  for (int g = 0; g < 2; g++)
#pragma unroll
    for (int n = 0; n < kTiles; n++) acc[g][n] = f32x4{0, 0, 0, 0};
#pragma unroll
  for (int i0 = 0; i0 < NG; i0 += kRun) {
    // past the codes' end the queries are zeros, and any number will do
    const int w = min(Order<NG>::dword(i0, quad), kRun == 1 ? W - 1 : 4 * NG - kRun);
    uint32_t x[2][kRun];
    float scale[2];
#pragma unroll
    for (int g = 0; g < 2; g++) {
      __builtin_memcpy(x[g], __builtin_assume_aligned(&lds.codes[0][row + 16 * g][w], 4 * kRun),
                       4 * kRun);
      scale[g] = scale_of(lds.scales[0][w >> 2][at + col + 16 * g]);
    }
#pragma unroll
    for (int i = 0; i < kRun; i++)
#pragma unroll
      for (int g = 0; g < 2; g++) {
        const bf16x8 k = codes8_bf16(x[g][i], scale[g]);
#pragma unroll
        for (int n = 0; n < kTiles; n++)
#pragma unroll
          for (int m = 0; m < QueryTerms<T>::n; m++)
            acc[g][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[n].terms[m][i0 + i],
                                                                acc[g][n], 0, 0, 0);
      }
  }
}

// A lane's part of the values of 32 tokens from row `at` of LDS on: dword `w` of the codes of
// tokens 4 quad + r and 16 + 4 quad + r, and their scales' bytes, four to a dword.
struct Values {
  uint32_t codes[8];
  uint32_t scales[2];

  template <typename Lds>
  __device__ __forceinline__ void load(const Lds& lds, int at, int quad, int w) {
#pragma unroll
    for (int k = 0; k < 8; k++) codes[k] = lds.codes[1][at + 16 * (k >> 2) + 4 * (k & 3) + quad][w];
#pragma unroll
    for (int g = 0; g < 2; g++)
      scales[g] =
          *reinterpret_cast<const uint32_t*>(&lds.scales[1][w >> 2][at + 16 * g + 4 * quad]);
  }

  __device__ __forceinline__ void to_f32(float (&scale)[8]) const {
#pragma unroll
    for (int k = 0; k < 8; k++) scale[k] = scale_of((scales[k >> 2] >> (8 * (k & 3))) & 255);
  }
};

// Scales from 2^126 on, and the one of a group without a number: a code times such a scale may be
// no finite number, which times the weight 0 of a row that does not see the token is NaN. Such
// groups of V are kept out of the products' operands (tame) and added by hand to the rows that see
// their token (add_wild).
constexpr uint32_t kWildByte = 253;
constexpr float kWildScale = 0x1p126f;  // as scale_of has it

// Eight tokens' codes and scales without the wild ones.
__device__ __forceinline__ void tame(uint32_t (&codes)[8], float (&scale)[8]) {
#pragma unroll
  for (int k = 0; k < 8; k++) {
    const bool wild = scale[k] >= kWildScale;
    codes[k] = wild ? 0 : codes[k];
    scale[k] = wild ? 1.0f : scale[k];
  }
}

// A value at a device address that is a multiple of four; an address out of LDS must say so, or the
// load counts as one that may be of LDS and is waited for with those.
template <typename T>
__device__ __forceinline__ T load_global(uint64_t p) {
  typedef T Packed __attribute__((aligned(4)));
  return *reinterpret_cast<const __attribute__((address_space(1))) Packed*>(p);
}

// ---------------------------------------------------------------- the cache's rows, through LDS
// A workgroup's waves together fetch the K and V rows of a stage: kPairs (token, head)
// pairs a wave, token by token (heads that lie side by side in memory are read side by side), each
// row as 16-byte chunks and its scale dwords, into registers a stage ahead of their use, then into
// LDS. There the rows of a head follow one another, and the scale bytes of a group of its tokens.

//
// kWhole: the codes are whole chunks (the dwords of a half-row's codes are a multiple of four).
template <int NG, int kPairs, int kWaves, bool kWhole>
struct Stage {
  static constexpr int kLoads = (kPairs * NG + 63) / 64;  // of chunks, for K and for V
  static constexpr int kScaleDwords = NG > 4 ? 2 : 1;
  static constexpr int kRowDwords = 4 * NG;
  static constexpr int kRowsOf = kPairs * kWaves;  // (token, head) pairs

  struct Lds {
    alignas(16) uint32_t codes[2][kRowsOf][kRowDwords];
    alignas(16) uint8_t scales[2][NG][kRowsOf];
  };
  // Addresses of the stage's tokens' rows and whether they are tokens, ahead of the stage.
  struct Tokens {
    uint64_t at[4][kRowsOf];
    uint32_t ok[8][kRowsOf / 32];
    uint32_t wild[4][kWaves];  // the V rows that a wave fetched may hold a wild group (kWildByte)
  };

  // A chunk's token in the stage (8 bits), the dword of it in the cache from the token's first head
  // on (10 bits: see `deal` on heads that lie side by side) and its dword in LDS (13 bits).
  uint32_t chunk[kLoads];
  uint32_t last;  // the same of the lane's scales, with their row in LDS
  u32x4 codes[2][kLoads];
  uint32_t scale[kScaleDwords];
  static_assert(kRowsOf <= 256 && kRowsOf * kRowDwords <= 1 << 13, "");

  static __device__ __forceinline__ uint32_t pack(uint32_t token, uint32_t from, uint32_t to) {
    return token | (from << 8) | (to << 18);
  }
  static __device__ __forceinline__ uint32_t token_of(uint32_t x) { return x & 255; }
  static __device__ __forceinline__ uint32_t from_of(uint32_t x) { return (x >> 8) & 1023; }
  static __device__ __forceinline__ uint32_t to_of(uint32_t x) { return x >> 18; }

  // The stage has `tokens` tokens of `held.d` heads.
  __device__ __forceinline__ void place(const AttendArgs& a, int wave, int lane,
                                        const FastDiv& held, uint32_t tokens) {
    const uint32_t head_dwords = held.d > 1 ? static_cast<uint32_t>(a.c.sh) >> 2 : 0;
    uint32_t token, h;
#pragma unroll
    for (int j = 0; j < kLoads; j++) {
      const uint32_t i = j * 64 + lane;
      const uint32_t pair = min(i / NG, kPairs - 1u) + kPairs * wave, c = min(i % NG, a.c.NG - 1u);
      held.divmod(pair, token, h);
      // the last chunk moves back where it would pass the codes' end
      const uint32_t dword = max(min(4 * static_cast<int>(c), a.c.W - 4), 0);
      chunk[j] = pack(token, h * head_dwords + dword,
                      (h * tokens + place_of(token)) * kRowDwords + dword);
    }
    // scales: pairs of K, then of V
    held.divmod(lane % kPairs + kPairs * wave, token, h);
    last = pack(token, h * head_dwords + a.c.W, h * tokens + token);
  }

  __device__ __forceinline__ void fetch(const AttendArgs& a, const uint64_t* at, int lane) {
    // sums with the offsets, and those widened to 64 bits, are not to be kept in registers
    uint64_t skv = static_cast<uint64_t>(a.c.skv);
    asm volatile("" : "+s"(skv));
#pragma unroll
    for (int j = 0; j < kLoads; j++) {
      uint32_t x = chunk[j];
      asm volatile("" : "+v"(x));
      const uint64_t p = at[token_of(x)] + 4 * from_of(x);
#pragma unroll
      for (int kv = 0; kv < 2; kv++) {
        const uint64_t from = kv ? p + skv : p;
        if (NG == 2 && !kWhole && a.c.W == 2) {  // a row of 12 bytes
          codes[kv][j][0] = load_global<uint32_t>(from);
          codes[kv][j][1] = load_global<uint32_t>(from + 4);
        } else {
          codes[kv][j] = load_global<u32x4>(from);
        }
      }
    }
    uint32_t x = last;
    asm volatile("" : "+v"(x));
    const uint64_t p = at[token_of(x)] + 4 * from_of(x) + (lane & kPairs ? skv : 0);
#pragma unroll
    for (int k = 0; k < kScaleDwords; k++) scale[k] = load_global<uint32_t>(p + 4 * k);
  }

  __device__ __forceinline__ void store(const AttendArgs& a, Lds& lds, Tokens& t, int stage,
                                        int wave, int lane) {
#pragma unroll
    for (int j = 0; j < kLoads; j++) {
      // lanes past the chunks write again what the last of them does
      uint32_t x = chunk[j];
      asm volatile("" : "+v"(x));
#pragma unroll
      for (int kv = 0; kv < 2; kv++) {
        uint32_t* p = &lds.codes[kv][0][0] + to_of(x);
        if (kWhole) {
          *reinterpret_cast<u32x4*>(p) = codes[kv][j];
        } else {
#pragma unroll
          for (int k = 0; k < 4; k++) p[k] = codes[kv][j][k];
        }
      }
    }
    uint32_t y = last;
    asm volatile("" : "+v"(y));
    const uint32_t row = to_of(y);
    const int kv = lane & kPairs ? 1 : 0;
    const bool ok = (t.ok[stage & 7][token_of(y) >> 5] >> (y & 31)) & 1;
    bool wild = false;
#pragma unroll
    for (int k = 0; k < kScaleDwords; k++) {
      // a token outside the context must be a number, whatever its row holds: its weight is 0
      const uint32_t x = ok ? scale[k] : 0x7F7F7F7Fu;
      // a byte of ~x is below 3 (or a 3 above such a byte)
      wild |= ((~x - 0x03030303u) & x & 0x80808080u) != 0;
#pragma unroll
      for (int g = 4 * k; g < NG && g < 4 * k + 4; g++)
        lds.scales[kv][g][row] = static_cast<uint8_t>(x >> (8 * (g & 3)));
    }
    const bool any = __builtin_amdgcn_ballot_w64(wild && kv) != 0;
    if (lane == 0) t.wild[stage & 3][wave] = any;
  }

  // The page of the thread's token of a stage, read a stage before its address is needed. (No
  // branch stands around this load or those of `fetch`, or the compiler loses count of the loads
  // under way and waits for all of them.)
  static __device__ __forceinline__ int32_t page_of(const AttendArgs& a, const int32_t* table,
                                                    uint32_t t, uint32_t stop) {
    return table[a.c.div_bs.div(min(t, stop - 1))];
  }

  // The tokens' addresses and flags, by as many threads.
  static __device__ __forceinline__ void locate(const AttendArgs& a, Tokens& s, int stage,
                                                const char* base, uint32_t t, uint32_t stop,
                                                int32_t page, uint32_t tid, uint32_t tokens) {
    const bool ok = tid < tokens && t < stop && page >= 0 && page < a.c.num_blocks;
    uint32_t q, off;
    a.c.div_bs.divmod(min(t, stop - 1), q, off);
    const unsigned long long flags = __builtin_amdgcn_ballot_w64(ok);
    if (tid < tokens) {
      s.at[stage & 3][tid] = reinterpret_cast<uint64_t>(base) +
                             (ok ? page * a.c.sb + static_cast<int64_t>(off) * a.c.so : 0);
      if ((tid & 31) == 0) s.ok[stage & 7][tid >> 5] = static_cast<uint32_t>(flags >> (tid & 32));
    }
  }
};

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

// Whether eight new scores of each of this lane's rows (masked ones -infinity) take some row's
// maximum too far past its reference: then all sums so far must be multiplied by `fade`.
template <int kTiles>
__device__ __forceinline__ bool grow(const float (&s)[kTiles][8], float scale_log2,
                                     Running (&r)[kTiles], float (&fade)[kTiles]) {
  float top[kTiles];
  bool far = false;
#pragma unroll
  for (int n = 0; n < kTiles; n++) {
    float x = s[n][0];
#pragma unroll
    for (int k = 1; k < 8; k++) x = fmaxf(x, s[n][k]);
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

// Eight scores of this lane's row to weights.
template <int kTerms>
__device__ __forceinline__ void weights(const float (&s)[8], float scale_log2, Running& r,
                                        u32x4 (&p)[kTerms]) {
  const float shift = r.shift();
#pragma unroll
  for (int k = 0; k < 8; k += 2) {
    const float lo = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k], scale_log2, -shift));
    const float hi = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k + 1], scale_log2, -shift));
    r.l += lo + hi;
    const uint32_t w = pack_bf16(lo, hi);
    p[0][k / 2] = w;
    if (kTerms > 1)
      p[kTerms - 1][k / 2] = pack_bf16(lo - __builtin_bit_cast(float, w << 16),
                                       hi - __builtin_bit_cast(float, w & 0xFFFF0000u));
  }
}

// The products of the wild groups of V (kWildByte) among the 32 tokens from row `at` of LDS, whose
// scores for this lane's row are `s`: the lane's elements of o[j][r] (dword 16 v + 4 quad + r, one
// group) get them if its row sees the token. `ahead` counts from the first of the 32.
template <typename Lds>
__device__ __forceinline__ void add_wild(const Lds& lds, int at, int v, int W, int ahead,
                                         uint32_t ok, const float (&s)[8], float scale_log2,
                                         const Running& r, f32x4 (&o)[8]) {
  const int lane = lane_now();
  const int quad = lane >> 4, w0 = 16 * v + 4 * quad;
  Running now = r;  // its shift is not to be shared with the weights', on the way of all stages
  asm volatile("" : "+v"(now.m));
  const float shift = now.shift();
#pragma unroll 1
  for (int k = 0; k < 32; k++) {
    // the token's score is with the lanes of quarter k / 4 % 4
    float mine = s[0];
#pragma unroll
    for (int i = 1; i < 8; i++) mine = 4 * (k >> 4) + (k & 3) == i ? s[i] : mine;
    mine = __shfl(mine, (lane & 15) + 16 * ((k >> 2) & 3));
    const uint32_t byte = lds.scales[1][min(w0, W - 1) >> 2][at + k];
    if (byte < kWildByte || k > ahead || !((ok >> k) & 1)) continue;
    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(mine, scale_log2, -shift));
    const float scale = scale_of(byte);
    const uint32_t* row = lds.codes[1][at + place_of(k)];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t x = row[min(w0 + i, W - 1)];
      const auto pair = [&](int c, f32x2 value) {
        o[2 * c][i] += p * value[0];
        o[2 * c + 1][i] += p * value[1];
      };
      pair(0, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x, scale, 0));
      pair(1, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x, scale, 1));
      pair(2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x, scale, 2));
      pair(3, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x, scale, 3));
    }
  }
}

// Dword codes of eight tokens and their scales to the operands of the products of elements 2c and
// 2c + 1 of each dword.
template <int c>
__device__ __forceinline__ void value_pair(const uint32_t (&x)[8], const float (&scale)[8],
                                           bf16x8& even, bf16x8& odd) {
  u32x4 e, o;
#pragma unroll
  for (int k = 0; k < 8; k += 2) {
    const uint32_t a = codes_bf16<c>(x[k], scale[k]);
    const uint32_t b = codes_bf16<c>(x[k + 1], scale[k + 1]);
    e[k / 2] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    o[k / 2] = __builtin_amdgcn_perm(b, a, 0x07060302u);
  }
  even = __builtin_bit_cast(bf16x8, e);
  odd = __builtin_bit_cast(bf16x8, o);
}

// ---------------------------------------------------------------- results
// One dword's eight elements of an output row, from the sums, their reference and the weights'
// total.
template <typename T>
__device__ __forceinline__ void finish(const AttendArgs& a, const Sequence& sq, int row,
                                       uint32_t head, int w, const float (&v)[8], float top,
                                       float total) {
  const float inv = total > 0 ? 1.0f / total : (total == 0 ? 0.0f : total);  // NaN stays
  uint32_t i, g;
  a.shared.divmod(row, i, g);
  const int64_t at = static_cast<int64_t>(sq.q0 + i) * a.q_heads + head * a.shared.d + g;
  T y[8];
#pragma unroll
  for (int j = 0; j < 8; j++) y[j] = static_cast<T>(v[j] * inv);
  __builtin_memcpy(__builtin_assume_aligned(a.out + (at * a.c.W + w) * 16, 16), y, 16);
  if (w == 0 && a.lse != nullptr)
    a.lse[at] = total == 0 ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * kLn2;
}

// Where a part's row of a head lies; such rows start on 8 bytes.
__device__ __forceinline__ float* part_row(const AttendArgs& a, const Dealt& dealt, uint32_t owner,
                                           uint32_t slot, uint32_t head, int r) {
  return dealt.part + ((static_cast<int64_t>(owner) * 2 + slot) * a.c.heads + head) *
                          (static_cast<int64_t>(dealt.rows) * (a.c.d + 2)) +
         static_cast<int64_t>(r) * (a.c.d + 2);
}

// A dword's eight sums of a part's row, for the join.
__device__ __forceinline__ void keep(const AttendArgs& a, float* part, int w, const float (&v)[8],
                                     float top, float total) {
  __builtin_memcpy(__builtin_assume_aligned(part + 8 * w, 8), v, sizeof(v));
  if (w == 0) {
    part[a.c.d] = top;
    part[a.c.d + 1] = total;
  }
}

// For the join, by one thread of the share with the tile's start.
template <bool kMany>
__device__ __forceinline__ void describe(const AttendArgs& a, const Share& r, uint32_t owner,
                                         const Part& p) {
  const Dealt& dealt = kMany ? a.many : a.few;
  const uint32_t first = static_cast<uint32_t>((r.line + kStart<kMany>) / r.size);
  const uint32_t last = static_cast<uint32_t>((r.line + p.places - 1) / r.size);
  const uint32_t parts = last - first + 1;
  if (kMany)
    dealt.tiles_in[owner] = make_uint4(r.seq, r.tile, parts, 0);
  else
    dealt.tiles_in[static_cast<int64_t>(r.seq) * dealt.most.d + r.tile] =
        make_uint4(first, parts, 0, 0);
}

int attend_few(const AttendArgs& a, int type, hipStream_t s);
int attend_many(const AttendArgs& a, int type, hipStream_t s);

}  // namespace evs
