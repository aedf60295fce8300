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
constexpr int kRows = 16;              // query rows of a tile
constexpr int kTile = 32;              // tokens a wave takes at once
constexpr int kSpan = kWaves * kTile;  // tokens a workgroup's waves take at once
constexpr uint32_t kMinSpans = 4;      // the fewest spans of a split
constexpr int64_t kWorkgroups = 2048;  // workgroups that a call's splits aim at
constexpr float kLn2 = 0.6931471805599453f;

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
  FastDiv shared;    // query heads that share a KV head
  FastDiv heads;
  float scale_log2;  // scale * log2(e)
  uint32_t units;    // workgroups a KV head has, a multiple of 8
  uint32_t tiles;    // row tiles a KV head may have
  uint32_t tile_rows;  // rows of them that are ever used
  bool split;        // a context may be split over several of them
  uint32_t join_bits;  // log2 of a joined row's dwords, rounded up
  float* part;       // [units, heads, kRows, d + 2]: a split's sums, running maximum and total
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

// A workgroup's share: split `split` of `splits` of row tile `tile` of sequence `seq`.
struct Unit {
  int32_t seq, tile, split, splits, step;
  uint32_t first;  // the unit of split 0
};

template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

// The units are the splits of the row tiles of the sequences, in that order. With splits, a split
// is the fewest spans of tokens with which all of them fit in `units`: with `total` spans over all
// tiles and `base` tiles, ceil(total / (units - base)) spans give at most total / that + base
// splits. Every workgroup finds its unit by itself from the lengths, so nothing is planned ahead of
// the launch. False: no unit is left for it.
//
// kTiles: `unit` counts row tiles instead, and the tile's first unit is found.
template <bool kTiles = false>
__device__ __forceinline__ bool find_unit(const AttendArgs& a, uint32_t unit, Unit& u) {
  __shared__ unsigned long long s_total[kWaves];
  __shared__ uint32_t s_base[kWaves];
  __shared__ int32_t s_unit[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  u.step = 0x7FFFFFFF;
  if (a.split) {
    unsigned long long total = 0;
    uint32_t base = 0;
    for (int s = tid; s < a.seqs; s += kThreads) {
      const Sequence q = sequence(a, s);
      const uint32_t tiles = (q.rows + kRows - 1) / kRows;
      base += tiles;
      total += static_cast<unsigned long long>(tiles) * ((q.len + kSpan - 1u) / kSpan);
    }
    total = wave_sum(total);
    base = wave_sum(base);
    if (lane == 0) {
      s_total[wave] = total;
      s_base[wave] = base;
    }
    __syncthreads();
    total = 0;
    base = 0;
#pragma unroll
    for (int k = 0; k < kWaves; k++) {
      total += s_total[k];
      base += s_base[k];
    }
    const uint32_t room = a.units > base ? a.units - base : 1;
    const unsigned long long spans = (total + room - 1) / room;
    const uint32_t few = spans < kMinSpans ? kMinSpans : static_cast<uint32_t>(spans);
    u.step = few > 0x7FFFFFFFu / kSpan ? 0x7FFFFFFF : static_cast<int32_t>(few * kSpan);
    __syncthreads();
  }
  if (tid == 0) s_unit[0] = -1;
  uint32_t before = 0, tiles_before = 0;
  for (int s0 = 0; s0 < a.seqs; s0 += kThreads) {
    const int s = s0 + tid;
    uint32_t tiles = 0, splits = 1;
    if (s < a.seqs) {
      const Sequence q = sequence(a, s);
      tiles = (q.rows + kRows - 1) / kRows;
      if (q.len > u.step) splits = (q.len + u.step - 1u) / static_cast<uint32_t>(u.step);
    }
    const uint32_t mine = tiles * splits;
    uint32_t sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t up = __shfl_up(sum, d);
      if (lane >= d) sum += up;
    }
    if (lane == 63) s_base[wave] = sum;
    __syncthreads();
    uint32_t start = before + sum - mine, all = 0;
#pragma unroll
    for (int k = 0; k < kWaves; k++) {
      if (k < wave) start += s_base[k];
      all += s_base[k];
    }
    if constexpr (kTiles) {
      // the same over the tiles
      uint32_t t_sum = tiles;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const uint32_t up = __shfl_up(t_sum, d);
        if (lane >= d) t_sum += up;
      }
      __syncthreads();
      if (lane == 63) s_base[wave] = t_sum;
      __syncthreads();
      uint32_t t_start = tiles_before + t_sum - tiles, t_all = 0;
#pragma unroll
      for (int k = 0; k < kWaves; k++) {
        if (k < wave) t_start += s_base[k];
        t_all += s_base[k];
      }
      if (unit >= t_start && unit - t_start < tiles) {
        s_unit[0] = s;
        s_unit[1] = static_cast<int32_t>((unit - t_start) * splits);
        s_unit[2] = static_cast<int32_t>(splits);
        s_unit[3] = static_cast<int32_t>(start + (unit - t_start) * splits);
      }
      tiles_before += t_all;
    } else if (unit >= start && unit - start < mine) {
      s_unit[0] = s;
      s_unit[1] = static_cast<int32_t>(unit - start);
      s_unit[2] = static_cast<int32_t>(splits);
    }
    before += all;
    __syncthreads();
    if (unit < (kTiles ? tiles_before : before)) break;
  }
  __syncthreads();
  u.seq = __builtin_amdgcn_readfirstlane(s_unit[0]);
  if (u.seq < 0) return false;
  u.splits = __builtin_amdgcn_readfirstlane(s_unit[2]);
  const int32_t at = __builtin_amdgcn_readfirstlane(s_unit[1]);
  u.tile = at / u.splits;
  u.split = at - u.tile * u.splits;
  u.first = kTiles ? __builtin_amdgcn_readfirstlane(s_unit[3]) : unit - u.split;
  return true;
}

template <typename T>
struct QueryTerms;  // bf16 terms that a query, and a weight for such a query's output, is the sum of
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

__device__ __forceinline__ uint32_t load_byte(const char* p) {
  return *reinterpret_cast<const uint8_t*>(p);
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

// One dword's eight elements of an output row, from the sums, their reference and the weights' total.
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

// How the pages' rows are found. kByTile: 16 tokens from a multiple of 16 lie in one page (its size
// is a multiple of 16), whose id is read once for the wave; kByToken: every token by itself.
enum Paging { kByTile, kByToken };

// What a wave holds of 32 tokens before it computes with them.
template <int NW, int VD, int NB>
struct Tokens {
  Dwords<NW> kc[2];        // K's codes of token 16 g + col, this quarter's dwords
  uint32_t ks[2][NB];      // and the scale bytes they have
  uint32_t vc[VD][8];      // V's codes of tokens 16 g + 4 quad + r, dword 16 v + col
  uint32_t vs[VD][8];      // and their scale bytes
  uint32_t bad;            // bit 8: this lane's V token has no page (and bits 0 to 7: which)
};

// One workgroup: a split of a tile of 16 query rows of one KV head of one sequence. Each of its
// waves takes a quarter of the split's tokens, 32 at a time, the next 32 being loaded meanwhile,
// and they join their results in LDS.
//
// NW: dwords of codes of K that a quarter of a wave's lanes holds; VD: dwords of V a lane holds.
// AL: those NW dwords have NW / 4 scales, or one (head sizes 64, 128 and 256).
template <int NW, int VD, bool AL, Paging P, typename T>
__global__ __launch_bounds__(kThreads, VD == 1 ? 3 : 2) void attend_rows(AttendArgs a) {
  constexpr int kTerms = QueryTerms<T>::n;
  constexpr int kDims = 128 * VD;  // the output tile's width, its padding included
  constexpr int NB = AL ? (NW + 3) / 4 : (NW + 2) / 4 + 1;
  __shared__ float s_o[kWaves][kRows][kDims + 4];
  __shared__ float s_m[kWaves][kRows];
  __shared__ float s_l[kWaves][kRows];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  // Workgroups go to the 8 XCDs in turn: a unit's heads, whose rows share memory lines, to one.
  uint32_t head, group;
  a.heads.divmod(blockIdx.x >> 3, group, head);
  const uint32_t unit = 8 * group + (blockIdx.x & 7);
  Unit u;
  if (!find_unit(a, unit, u)) return;
  const Sequence sq = sequence(a, u.seq);
  const int row0 = u.tile * kRows;
  const int last_row = min(row0 + kRows, sq.rows) - 1;

  // this lane's query row, and the tokens that it sees: those up to `sees`
  const int row = min(row0 + col, last_row);
  uint32_t qi, qg;
  a.shared.divmod(row, qi, qg);
  const int past = sq.len - sq.nq;
  const int sees = past + static_cast<int>(qi);
  // tokens that some row sees, and those that all of them see
  const int end = min(sq.len, past + static_cast<int>(a.shared.div(last_row)) + 1);
  const int all_see = min(end, past + static_cast<int>(a.shared.div(row0)) + 1);
  const int begin = u.split == 0 ? 0 : u.split * u.step;
  const int stop = u.splits == 1 ? end : min(end, begin + u.step);

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
  const int32_t* table = a.tables + static_cast<int64_t>(u.seq) * a.table_stride;
  // this lane's places within 16 tokens' rows of K and V
  const uint32_t so = static_cast<uint32_t>(a.c.so);  // kByTile: 16 of them are below 2^31
  const uint32_t k_at = col * so + 4 * w0;
  uint32_t v_at[VD];
  int vw[VD];
#pragma unroll
  for (int v = 0; v < VD; v++) {
    vw[v] = min(16 * v + col, W - 1);
    v_at[v] = 4 * quad * so + 4 * vw[v];
  }
  const int ks0 = w0 >> 2;  // this quarter's first scale

  // The pages of 16 tokens from t on, and their first row there; kByTile alone.
  struct Page {
    int32_t id[2];
  };
  const auto pages_at = [&](int t) {
    Page p;
#pragma unroll
    for (int g = 0; g < 2; g++) {
      const int tg = t + 16 * g;
      p.id[g] = tg < stop ? table[a.c.div_bs.div(tg)] : -1;
      if (p.id[g] >= a.c.num_blocks) p.id[g] = -1;
    }
    return p;
  };
  const auto row_of = [&](int t, bool& ok) {
    uint32_t page, off;
    a.c.div_bs.divmod(min(t, stop - 1), page, off);
    const int32_t block = table[page];
    ok = t < stop && block >= 0 && block < a.c.num_blocks;
    return base + (ok ? block : 0) * a.c.sb + off * a.c.so;
  };

  typedef Tokens<NW, VD, NB> Held;
  const auto load = [&](Held& h, int t, const Page& pg) {
    h.bad = 0;
#pragma unroll
    for (int g = 0; g < 2; g++) {
      const char *kp, *vp[4];
      if constexpr (P == kByTile) {
        const int tg = t + 16 * g;
        const uint32_t off = tg - a.c.div_bs.div(tg) * a.c.block_size;
        const char* rows = base + max(pg.id[g], 0) * a.c.sb + static_cast<int64_t>(off) * a.c.so;
        kp = rows;
        if (pg.id[g] < 0) h.bad |= 0x10F << (4 * g);
#pragma unroll
        for (int r = 0; r < 4; r++) vp[r] = rows + a.c.skv + static_cast<int64_t>(r) * a.c.so;
      } else {
        bool ok;
        kp = row_of(t + 16 * g + col, ok) + 4 * w0;
#pragma unroll
        for (int r = 0; r < 4; r++) {
          vp[r] = row_of(t + 16 * g + 4 * quad + r, ok) + a.c.skv;
          if (!ok) h.bad |= 0x100 | (1 << (4 * g + r));
        }
      }
      const uint32_t ko = P == kByTile ? k_at : 0;
      h.kc[g] = load_dwords<NW>(kp + ko);
#pragma unroll
      for (int b = 0; b < NB; b++) {
        const int sb = AL ? ks0 + b : min(ks0 + b, a.c.NG - 1);
        h.ks[g][b] = load_byte(kp + (ko - (P == kByTile ? 4 * w0 : 0)) +
                               (4 * W + sb - (P == kByTile ? 0 : 4 * w0)));
      }
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int v = 0; v < VD; v++) {
          const uint32_t vo = P == kByTile ? v_at[v] : 4 * vw[v];
          h.vc[v][4 * g + r] = load_dwords<1>(vp[r] + vo).v[0];
          h.vs[v][4 * g + r] = load_byte(vp[r] + (vo - 4 * vw[v] + 4 * W + (vw[v] >> 2)));
        }
    }
  };

  f32x4 o[VD][8];
#pragma unroll
  for (int v = 0; v < VD; v++)
#pragma unroll
    for (int j = 0; j < 8; j++) o[v][j] = f32x4{0, 0, 0, 0};
  // This lane's row's reference for its weights (scaled scores), the same for its four lanes; the
  // maximum seen is at most kSlack above it. And this lane's part of the weights' sum.
  constexpr float kSlack = 8.0f;
  float m = -INFINITY, shift = 0.0f, l = 0.0f;

  const auto compute = [&](const Held& h, int t) {
    f32x4 acc[2];
#pragma unroll
    for (int g = 0; g < 2; g++) {
      acc[g] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < NW; i++) {
        uint32_t byte = h.ks[g][AL ? i / 4 : 0];
        if constexpr (!AL) {
          const int at = ((w0 + i) >> 2) - ks0;
#pragma unroll
          for (int b = 1; b < NB; b++) byte = at == b ? h.ks[g][b] : byte;
        }
        const bf16x8 k = codes8_bf16(h.kc[g].v[i], scale_of(byte));
#pragma unroll
        for (int n = 0; n < kTerms; n++)
          acc[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, qf[n][i], acc[g], 0, 0, 0);
      }
    }
    float s[8];
#pragma unroll
    for (int k = 0; k < 8; k++) s[k] = acc[k >> 2][k & 3];
    uint32_t bad = h.bad;
    const bool whole =
        t + kTile <= min(stop, all_see) &&
        (P == kByTile ? bad == 0 : __builtin_amdgcn_ballot_w64(bad != 0) == 0);
    if (!whole) {
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const int tk = t + 16 * (k >> 2) + 4 * quad + (k & 3);
        if (tk >= stop) bad |= 1u << k;
        s[k] = tk <= sees && !((bad >> k) & 1) ? s[k] : -INFINITY;
      }
    }
    float top = s[0];
#pragma unroll
    for (int k = 1; k < 8; k++) top = fmaxf(top, s[k]);
    top *= a.scale_log2;
    if (__builtin_amdgcn_ballot_w64(top > m + kSlack) != 0) {
      top = fmaxf(across_rows_max(top), m);
      const float now = top == -INFINITY ? 0.0f : top;  // a row that has seen nothing yet
      const float fade = __builtin_amdgcn_exp2f(m - now);
      m = top;
      shift = now;
      l *= fade;
#pragma unroll
      for (int v = 0; v < VD; v++)
#pragma unroll
        for (int j = 0; j < 8; j++) o[v][j] *= fade;
    }
    u32x4 p[kTerms];
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
      const float lo = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k], a.scale_log2, -shift));
      const float hi = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k + 1], a.scale_log2, -shift));
      l += lo + hi;
      const uint32_t w = pack_bf16(lo, hi);
      p[0][k / 2] = w;
      if (kTerms > 1)
        p[kTerms - 1][k / 2] = pack_bf16(lo - __builtin_bit_cast(float, w << 16),
                                         hi - __builtin_bit_cast(float, w & 0xFFFF0000u));
    }
#pragma unroll
    for (int v = 0; v < VD; v++) {
      float sc[8];
#pragma unroll
      for (int k = 0; k < 8; k++) sc[k] = scale_of(h.vs[v][k]);
      // a token outside the context must be a number, whatever its row holds: its weight is 0
      if (!whole) {
#pragma unroll
        for (int k = 0; k < 8; k++) sc[k] = (bad >> k) & 1 ? 1.0f : sc[k];
      }
      // elements 2c and 2c + 1 of the eight tokens
      const auto pair = [&](auto c_) {
        constexpr int c = decltype(c_)::value;
        u32x4 even, odd;
#pragma unroll
        for (int k = 0; k < 8; k += 2) {
          const uint32_t x = codes_bf16<c>(h.vc[v][k], sc[k]);
          const uint32_t y = codes_bf16<c>(h.vc[v][k + 1], sc[k + 1]);
          even[k / 2] = __builtin_amdgcn_perm(y, x, 0x05040100u);
          odd[k / 2] = __builtin_amdgcn_perm(y, x, 0x07060302u);
        }
#pragma unroll
        for (int n = 0; n < kTerms; n++) {
          const bf16x8 pf = __builtin_bit_cast(bf16x8, p[n]);
          o[v][2 * c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, even),
                                                                pf, o[v][2 * c], 0, 0, 0);
          o[v][2 * c + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(bf16x8, odd), pf, o[v][2 * c + 1], 0, 0, 0);
        }
      };
      pair(std::integral_constant<int, 0>{});
      pair(std::integral_constant<int, 1>{});
      pair(std::integral_constant<int, 2>{});
      pair(std::integral_constant<int, 3>{});
    }
  };

  // The wave's tiles of 32 tokens: [first, last). Loads run a tile ahead, page ids two; past the
  // last tile it is read again, so that no branch stands between a load and its use.
  const int tiles = stop > begin ? (stop - begin + kTile - 1) / kTile : 0;
  const int first = wave * tiles / kWaves, last = (wave + 1) * tiles / kWaves;
  if (first < last) {
    const auto token = [&](int i) { return begin + kTile * min(i, last - 1); };
    Held even, odd;
    Page pg{};
    if constexpr (P == kByTile) pg = pages_at(token(first));
    load(even, token(first), pg);
    if constexpr (P == kByTile) pg = pages_at(token(first + 1));
    for (int i = first; i < last; i += 2) {
      load(odd, token(i + 1), pg);
      if constexpr (P == kByTile) pg = pages_at(token(i + 2));
      compute(even, token(i));
      if (i + 1 >= last) break;
      load(even, token(i + 2), pg);
      if constexpr (P == kByTile) pg = pages_at(token(i + 3));
      compute(odd, token(i + 1));
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
  for (int x = threadIdx.x; x < kRows * W; x += kThreads) {
    const int r = x / W, w = x - r * W;
    if (row0 + r > last_row) break;  // rows ascend
    float top = s_m[0][r];
#pragma unroll
    for (int k = 1; k < kWaves; k++) top = fmaxf(top, s_m[k][r]);
    const float ref = top == -INFINITY ? 0.0f : top;
    float total = 0, v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < kWaves; k++) {
      const float f = __builtin_amdgcn_exp2f(s_m[k][r] - ref);
      total += f * s_l[k][r];
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] += f * s_o[k][r][8 * w + j];
    }
    if (u.splits > 1) {
      float* part = a.part + ((static_cast<int64_t>(unit) * a.c.heads + head) * kRows + r) *
                                 (a.c.d + 2);
#pragma unroll
      for (int j = 0; j < 8; j++) part[8 * w + j] = v[j];
      if (w == 0) {
        part[a.c.d] = top;
        part[a.c.d + 1] = total;
      }
    } else {
      finish<T>(a, sq, row0 + r, head, w, v, top, total);
    }
  }
}

// One row of a row tile that was split, joined: one workgroup for each row tile (found as find_unit
// finds units), head and row. Its threads are dealt a dword of elements each and, several times
// over, the splits in turn.
template <typename T>
__global__ __launch_bounds__(kThreads) void join_splits(AttendArgs a) {
  __shared__ float s_v[kThreads][8 + 1];
  __shared__ float s_m[kThreads];
  __shared__ float s_l[kThreads];
  uint32_t head, tile;
  a.heads.divmod(blockIdx.x, tile, head);
  Unit u;
  if (!find_unit<true>(a, tile, u) || u.splits == 1) return;
  const Sequence sq = sequence(a, u.seq);
  const int row = u.tile * kRows + blockIdx.y;
  if (row >= sq.rows) return;
  // dwords of a row, rounded up to a power of two, times threads over the splits
  const uint32_t lanes = 1u << a.join_bits;
  const uint32_t w = threadIdx.x & (lanes - 1), turn = threadIdx.x >> a.join_bits;
  const uint32_t turns = kThreads >> a.join_bits;
  const int64_t row_floats = a.c.d + 2;
  const int64_t split_floats = a.c.heads * kRows * row_floats;
  const float* part =
      a.part + ((static_cast<int64_t>(u.first) * a.c.heads + head) * kRows + blockIdx.y) * row_floats;
  const uint32_t wr = min(w, static_cast<uint32_t>(a.c.W) - 1);
  float top = -INFINITY, total = 0, v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  for (uint32_t k = turn; k < static_cast<uint32_t>(u.splits); k += turns) {
    const float* p = part + k * split_floats;
    const float m = p[a.c.d], l = p[a.c.d + 1];
    float x[8];
    __builtin_memcpy(x, __builtin_assume_aligned(p + 8 * wr, 8), sizeof(x));
    const float now = fmaxf(top, m);
    const float ref = now == -INFINITY ? 0.0f : now;
    const float f = __builtin_amdgcn_exp2f(top - ref), g = __builtin_amdgcn_exp2f(m - ref);
    top = now;
    total = total * f + l * g;
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = v[j] * f + x[j] * g;
  }
  s_m[threadIdx.x] = top;
  s_l[threadIdx.x] = total;
#pragma unroll
  for (int j = 0; j < 8; j++) s_v[threadIdx.x][j] = v[j];
  __syncthreads();
  if (turn != 0 || w >= static_cast<uint32_t>(a.c.W)) return;
  const uint32_t some = min(turns, static_cast<uint32_t>(u.splits));
  for (uint32_t k = 1; k < some; k++) top = fmaxf(top, s_m[(k << a.join_bits) + w]);
  const float ref = top == -INFINITY ? 0.0f : top;
  total = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) v[j] = 0;
  for (uint32_t k = 0; k < some; k++) {
    const uint32_t t = (k << a.join_bits) + w;
    const float f = __builtin_amdgcn_exp2f(s_m[t] - ref);
    total += s_l[t] * f;
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] += s_v[t][j] * f;
  }
  finish<T>(a, sq, row, head, w, v, top, total);
}

template <int NW, int VD, bool AL, Paging P>
int launch(const AttendArgs& a, int type, hipStream_t s) {
  const uint32_t grid = a.units * static_cast<uint32_t>(a.c.heads);
  if (type == EVS_BF16)
    attend_rows<NW, VD, AL, P, __bf16><<<grid, kThreads, 0, s>>>(a);
  else
    attend_rows<NW, VD, AL, P, _Float16><<<grid, kThreads, 0, s>>>(a);
  EVS_LAUNCHED("evs_fp4_attend");
  if (a.split) {
    const dim3 rows(a.tiles * static_cast<uint32_t>(a.c.heads), a.tile_rows);
    if (type == EVS_BF16)
      join_splits<__bf16><<<rows, kThreads, 0, s>>>(a);
    else
      join_splits<_Float16><<<rows, kThreads, 0, s>>>(a);
    EVS_LAUNCHED("evs_fp4_attend");
  }
  return EVS_OK;
}

template <Paging P>
int launch_dims(const AttendArgs& a, int type, hipStream_t s) {
  switch (a.c.W) {
    case 8: return launch<2, 1, true, P>(a, type, s);
    case 16: return launch<4, 1, true, P>(a, type, s);
    case 32: return launch<8, 2, true, P>(a, type, s);
  }
  const int per = (a.c.W + 3) / 4;  // dwords of codes a quarter of the lanes holds
  if (per <= 2) return launch<2, 1, false, P>(a, type, s);
  if (per <= 3) return launch<3, 1, false, P>(a, type, s);
  if (per <= 4) return launch<4, 1, false, P>(a, type, s);
  if (per <= 6) return launch<6, 2, false, P>(a, type, s);
  return launch<8, 2, false, P>(a, type, s);
}

// How a call's work is dealt out, from its counts alone (the lengths are on the device).
struct Deal {
  int64_t units;  // for each KV head
  int64_t tiles;  // of rows, at most
  bool split;
  int64_t bytes;  // of the splits' workspace
};

Deal deal(int64_t seqs, int64_t tokens, int64_t shared, int64_t heads, int64_t d, int64_t max_q,
          int64_t max_len) {
  Deal r{};
  // row tiles: a sequence's rows, rounded up
  const int64_t most = (max_q * shared + kRows - 1) / kRows * seqs;
  const int64_t spread = tokens * shared / kRows + seqs;
  const int64_t base = most < spread ? most : spread;
  r.units = r.tiles = base;
  if (base * heads < kWorkgroups && max_len > kMinSpans * kSpan) {
    r.split = true;
    r.units += (kWorkgroups + heads - 1) / heads;
  }
  r.units = (r.units + 7) / 8 * 8;
  if (r.split) r.bytes = r.units * heads * kRows * (d + 2) * 4;
  return r;
}

}  // namespace
}  // namespace evs

extern "C" int evs_fp4_attend_workspace(int64_t seqs, int64_t tokens, int64_t q_heads,
                                        int64_t heads, int64_t head_dim, int64_t max_q,
                                        int64_t max_len, int64_t* bytes) {
  evs::clear_error();
  EVS_REQUIRE(bytes != nullptr, "evs_fp4_attend_workspace: null result");
  *bytes = 0;
  EVS_REQUIRE(seqs >= 0 && tokens >= 0 && max_q >= 0 && max_len >= 0 && heads > 0 &&
                  heads < (1 << 16) && q_heads > 0 && q_heads < (1 << 16) && q_heads % heads == 0 &&
                  seqs < (int64_t{1} << 31) && tokens < (int64_t{1} << 31) &&
                  head_dim <= evs::kFp4MaxDim,
              "evs_fp4_attend_workspace: bad count");
  if (seqs == 0 || tokens == 0 || max_q == 0) return EVS_OK;
  if (max_len == 0) max_len = INT64_MAX;
  *bytes = evs::deal(seqs, tokens, q_heads / heads, heads, head_dim, max_q < tokens ? max_q : tokens,
                     max_len)
               .bytes;
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
  if (max_len == 0 || max_len > width * block_size) max_len = width * block_size;
  const evs::Deal deal = evs::deal(seqs, tokens, shared, heads, head_dim, max_q, max_len);
  EVS_REQUIRE(deal.units * heads < (int64_t{1} << 24), "%s: %lld tiles of query rows: below 2^24",
              who, static_cast<long long>(deal.units * heads));
  EVS_REQUIRE(deal.bytes <= workspace_bytes &&
                  (deal.bytes == 0 || (workspace != nullptr &&
                                       reinterpret_cast<uintptr_t>(workspace) % 16 == 0)),
              "%s: a workspace of %lld bytes on 16, %lld needed", who,
              static_cast<long long>(workspace_bytes), static_cast<long long>(deal.bytes));
  a.units = static_cast<uint32_t>(deal.units);
  a.split = deal.split;
  a.tiles = static_cast<uint32_t>(deal.tiles);
  a.tile_rows = static_cast<uint32_t>(max_q * shared < evs::kRows ? max_q * shared : evs::kRows);
  while ((1 << a.join_bits) < a.c.W) a.join_bits++;
  a.part = static_cast<float*>(workspace);
  const hipStream_t s = evs::as_stream(stream);
  // the tile's rows are addressed in 32 bits from its first
  const bool by_tile = block_size % 16 == 0 && strides[1] >= 0 && strides[1] < (int64_t{1} << 26);
  return by_tile ? evs::launch_dims<evs::kByTile>(a, type, s)
                 : evs::launch_dims<evs::kByToken>(a, type, s);
}
