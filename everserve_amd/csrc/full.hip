// Attention over full-width pages: the calls, how their work is dealt out, and the join of contexts
// in several parts (full.hpp has the mathematics, full_attend.hip and full_weigh.hip the
// kernels).
#include "full.hpp"

namespace evs {
namespace {

// A row's parts, taken together: their maxima and totals.
__device__ __forceinline__ void join_stats(const float* stats, int64_t at, float& top,
                                           float& total) {
  const float m = stats[2 * at], l = stats[2 * at + 1];
  const float now = fmaxf(top, m);
  const float ref = now == -INFINITY ? 0.0f : now;
  total = total * __builtin_amdgcn_exp2f(top - ref) + l * __builtin_amdgcn_exp2f(m - ref);
  top = now;
}

// How the rows of a query are dealt to workgroups for the join: 2^words threads have four elements
// each of a row (or of a piece of it: `pieces` of them), 2^turns threads take the parts in turn, and
// the rest of a workgroup takes further heads; `down` workgroups take a query's heads and pieces.
struct JoinShape {
  int words, turns;
  FastDiv pieces, down;
};

// The rows of one query, joined from their parts.
template <typename T>
__device__ __forceinline__ void join_rows(const FullArgs& a, int token, int first,
                                          const JoinShape& shape) {
  __shared__ f32x4 s_v[kFullThreads];
  __shared__ float s_m[kFullThreads], s_l[kFullThreads];
  const int s = sequence_of(a, token);
  if (s < 0) return;  // uniform
  const Rows sq = scalar_rows(sequence_rows(a, s));
  const int shared = a.shared.d;
  // the prefix, and the own part of the context that a row's tile sees
  const bool few = sq.rows <= kRowTile, alone = sq.rows > kTogether;
  const Cut& cut = few ? a.few : a.many;
  if (!is_joined(a, cut, sq.rows, (1u << 31) - 1)) return;  // no row of it, however much it sees
  const int g = a.pre.n > 0 ? group_of(a, s) : -1;
  const int prefix = g < 0 ? 0 : length_of(a, a.pre, g);
  const int ahead = alone ? prefix : 0;
  const int tile = few ? kRowTile : kRowTile * kFullWaves * a.row_tiles;
  const int tid = threadIdx.x;
  const int mine = shape.words + shape.turns;
  const int heads_at = kFullThreads >> mine;
  const int turn = (tid >> shape.words) & ((1 << shape.turns) - 1);
  const int items = (a.q_heads + heads_at - 1) / heads_at * shape.pieces.d;
  for (int item = first; item < items; item += shape.down.d) {
    uint32_t at, piece;
    shape.pieces.divmod(item, at, piece);
    const int q_head = at * heads_at + (tid >> mine);
    const int in = min(q_head, a.q_heads - 1);
    const int w = (piece << shape.words) + (tid & ((1 << shape.words) - 1));
    const int wr = min(w, a.d / 4 - 1);
    const int head = in / shared, row = (token - sq.q0) * shared + in - head * shared;
    const int last = min(row / tile * tile + tile, sq.rows) - 1;
    const int end = min(ahead + sq.len, max(ahead + sq.len - sq.nq + last / shared + 1, ahead));
    const bool joined = q_head < a.q_heads && is_joined(a, cut, sq.rows, end);
    const int before = alone || !joined ? 0 : parts_of(a.group, prefix);
    const int parts = joined ? before + max(parts_of(cut, end), 1) : 0;
    float top = -INFINITY, total = 0;
    f32x4 v = {0, 0, 0, 0};
#pragma unroll 8
    for (int k = turn; k < parts; k += 1 << shape.turns) {
      const bool own = few && k >= before;
      const int64_t i = own ? few_part_at(a, k - before, s, head, row)
                            : part_at(a, k < before ? k : a.group.splits + k - before, token, in);
      const FullArgs::Parts& p = own ? a.few_parts : a.parts;
      const float m = p.stats[2 * i], l = p.stats[2 * i + 1];
      const f32x4 y = *reinterpret_cast<const f32x4*>(p.sums + i * a.d + 4 * wr);
      const float now = fmaxf(top, m);
      const float ref = now == -INFINITY ? 0.0f : now;
      const float f = __builtin_amdgcn_exp2f(top - ref), h = __builtin_amdgcn_exp2f(m - ref);
      top = now;
      total = total * f + l * h;
      v = v * f + y * h;
    }
    if (shape.turns > 0) {
      __syncthreads();  // the heads before have been read
      s_v[tid] = v;
      s_m[tid] = top;
      s_l[tid] = total;
      __syncthreads();
      if (turn == 0) {
        for (int k = 1; k < 1 << shape.turns; k++)
          top = fmaxf(top, s_m[tid + (k << shape.words)]);
        const float ref = top == -INFINITY ? 0.0f : top;
        total = 0;
        v = f32x4{0, 0, 0, 0};
        for (int k = 0; k < 1 << shape.turns; k++) {
          const int t = tid + (k << shape.words);
          const float f = __builtin_amdgcn_exp2f(s_m[t] - ref);
          total += s_l[t] * f;
          v += s_v[t] * f;
        }
      }
    }
    if (joined && turn == 0 && w < a.d / 4) finish4<T>(a, token, q_head, w, v, top, total);
  }
}

constexpr int kScored = 4 * kFullThreads;  // tokens of a workgroup

// The weights of a sequence with few rows, of one KV head and 1,024 of its own tokens, from the
// scores that the attention kept (full_weigh.hip has the formula and the other contexts). The rows'
// references are joined from the same parts as the rows, so it need not wait for those.
__device__ __forceinline__ void weigh_scores(const FullArgs& a, uint32_t seq, int head, int step) {
  __shared__ float s_top[kRowTile];
  constexpr int kAhead = 4;  // rows whose scores are on their way while the references are joined
  const Rows sq = scalar_rows(sequence_rows(a, seq));
  const int stop = min(sq.len, a.stored);
  const int t0 = step * kScored;
  if (sq.rows == 0 || sq.rows > kRowTile || t0 >= stop) return;
  const int tid = threadIdx.x, r = tid >> 4;
  const int past = sq.len - sq.nq;
  const int t = t0 + 4 * tid;
  const int in = min(t, (stop - 1) & ~3);
  const float* scores = a.scores + few_part_at(a, 0, seq, head, 0) * a.stored + in;
  const auto score = [&](int row) {
    return *reinterpret_cast<const f32x4*>(
        scores + static_cast<int64_t>(min(row, sq.rows - 1)) * a.stored);
  };
  f32x4 x[kAhead];
#pragma unroll
  for (int row = 0; row < kAhead; row++) x[row] = score(row);
  // where the tokens' masses are; null for no token
  const int32_t* table = a.own.tables + static_cast<int64_t>(seq) * a.own.stride;
  float* mass[4];
  float old[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    uint32_t n, off;
    a.div_bs.divmod(min(in + j, stop - 1), n, off);
    const int32_t page = table[n];
    mass[j] = t + j >= stop || page < 0 || page >= a.num_blocks
                  ? nullptr
                  : a.mass + (static_cast<int64_t>(page) * a.heads + head) * a.block_size + off;
  }
#pragma unroll
  for (int j = 0; j < 4; j++) old[j] = mass[j] == nullptr || t + j >= past ? 0.0f : *mass[j];
  {
    // 16 threads a row
    const int own = max(parts_of(a.few, sq.len), 1);
    const int g = a.pre.n > 0 ? group_of(a, seq) : -1;
    const int before = g < 0 || a.group.tiles == 0 ? 0 : parts_of(a.group, length_of(a, a.pre, g));
    float top = -INFINITY, total = 0;
    if (r < sq.rows) {
      uint32_t qi, qg;
      a.shared.divmod(r, qi, qg);
      for (int k = tid & 15; k < own; k += 16)
        join_stats(a.few_parts.stats, few_part_at(a, k, seq, head, r), top, total);
      for (int k = tid & 15; k < before; k += 16)
        join_stats(a.parts.stats, part_at(a, k, sq.q0 + qi, head * a.shared.d + qg), top, total);
    }
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
      const float m = __shfl_xor(top, d), l = __shfl_xor(total, d);
      const float now = fmaxf(top, m);
      const float ref = now == -INFINITY ? 0.0f : now;
      total = total * __builtin_amdgcn_exp2f(top - ref) + l * __builtin_amdgcn_exp2f(m - ref);
      top = now;
    }
    if ((tid & 15) == 0)
      s_top[r] = total == 0 ? INFINITY : top + __builtin_amdgcn_logf(total);
  }
  __syncthreads();
  f32x4 sum = {0, 0, 0, 0};
  const auto add = [&](int row, const f32x4& y) {
    const float top = s_top[row];
    const int sees = past + static_cast<int>(a.shared.div(row)) - t;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(y[j], a.scale_log2, -top));
      sum[j] += sees >= j && top != INFINITY ? w : 0.0f;
    }
  };
#pragma unroll
  for (int row = 0; row < kAhead; row++)
    if (row < sq.rows) add(row, x[row]);
#pragma unroll 4
  for (int row = kAhead; row < sq.rows; row++) add(row, score(row));
#pragma unroll
  for (int j = 0; j < 4; j++)
    if (mass[j] != nullptr) *mass[j] = old[j] + sum[j];
}

// The launch behind the attention's: the first workgroups join rows, the others weigh tokens by
// scores, `steps` of them a sequence and head.
template <typename T>
__global__ __launch_bounds__(kFullThreads) void join_full(FullArgs a, uint32_t join_items,
                                                          JoinShape shape, FastDiv steps) {
  if (blockIdx.x < join_items) {
    uint32_t token, first;
    shape.down.divmod(blockIdx.x, token, first);
    join_rows<T>(a, token, first, shape);
  } else {
    uint32_t rest, step, seq, head;
    steps.divmod(blockIdx.x - join_items, rest, step);
    a.div_heads.divmod(rest, seq, head);
    weigh_scores(a, seq, head, step);
  }
}

__global__ __launch_bounds__(kFullThreads) void no_weights(float* top, int64_t n) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kFullThreads + threadIdx.x;
  if (i < n) top[i] = INFINITY;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t least(int64_t a, int64_t b) { return a < b ? a : b; }

constexpr int64_t kRound = 256;  // tokens that a workgroup's waves take in turn, of few rows
constexpr int64_t kFillRows = 1024;
  // workgroups that fill the GPU, of few rows
constexpr int64_t kFillTiles = 256;  // and of many
// Beyond that, workgroups for few rows of contexts of unlike lengths, and the tokens of one.
constexpr int64_t kEven = 4096, kEvenChunk = 1024;
// A context of few rows without a prefix is one part up to here: a launch less than with parts that
// are joined. us of calls in a row, and replayed from a graph, on 8 KV heads of 128, in one part (and in
// parts of 256): one token over 600 11.5, 11.3 (12.4, 11.0), over 1,000 13.5, 13.4 (12.7, 11.4); 16
// sequences of 600 13.4, 13.5 (17.4, 17.2), of 1,000 16.5, 16.6 (20.1, 20.1). With mass the second
// launch follows either way and parts would be faster (one of 600 17.3 (12.9), 16 of 1,000 23.0 (20.5)),
// but a call gives the same bits with mass and without, so both are cut alike.
constexpr int64_t kBrief = 1024;
constexpr int64_t kWideGroup = 512;  // rows of small chunks, from which tiles of 128 are taken
constexpr int64_t kMostParts = 1024;
constexpr int64_t kMostScores = int64_t{1} << 29;  // bytes of scores that a call may keep

// How contexts of up to max_len tokens are cut for `tiles` row tiles that there may be: into parts
// that make `fill` workgroups in all, of `least_chunk` tokens at least, and beyond that into parts of
// `good_chunk` tokens that make `even` of them, so that contexts of unlike lengths end together.
Cut cut(int64_t tiles, int64_t heads, int64_t max_len, int64_t fill, int64_t least_chunk,
        int64_t even, int64_t good_chunk) {
  Cut c{};
  if (tiles == 0) return c;
  const int64_t parts_fill = least(ceil_div(fill, tiles * heads), ceil_div(max_len, least_chunk));
  const int64_t parts_even = least(ceil_div(even, tiles * heads), ceil_div(max_len, good_chunk));
  int64_t parts = parts_fill > parts_even ? parts_fill : parts_even;
  parts = parts < 1 ? 1 : least(parts, kMostParts);
  int64_t chunk = ceil_div(ceil_div(max_len, parts), kRound) * kRound;
  chunk = chunk < kRound ? kRound : least(chunk, (int64_t{1} << 31) - kRound);
  c.tiles = static_cast<uint32_t>(least(tiles, (int64_t{1} << 31) - 1));
  c.chunk = static_cast<int32_t>(chunk);
  c.splits = static_cast<int32_t>(least(ceil_div(max_len, chunk), kMostParts));
  if (c.splits < 1) c.splits = 1;
  return c;
}

struct Counts {
  int64_t seqs, tokens, q_heads, heads, d, max_q, max_len, groups, max_prefix;
  bool mass;
};

bool good(const Counts& n) {
  constexpr int64_t most = int64_t{1} << 31;
  return n.seqs >= 0 && n.seqs < most && n.tokens >= 0 && n.tokens < most && n.max_q >= 0 &&
         n.max_len >= 0 && n.groups >= 0 && n.groups < most && n.max_prefix >= 0 && n.heads > 0 &&
         n.heads < (1 << 16) && n.q_heads > 0 && n.q_heads < (1 << 16) &&
         n.q_heads % n.heads == 0 && n.d >= kFullMinDim && n.d <= kFullMaxDim && n.d % 8 == 0 &&
         n.tokens * (n.q_heads / n.heads) < most;
}

struct Deal {
  Cut group, few, many;
  bool few_groups;
  int row_tiles;
  int64_t slots, few_slots;  // of parts
  int64_t few_rows, stored;
  int64_t sums, stats, few_sums, few_stats, top, scores, bytes;
};

Deal deal(Counts n) {
  Deal r{};
  const int64_t shared = n.q_heads / n.heads;
  if (n.max_q > n.tokens) n.max_q = n.tokens;
  const int64_t most = n.max_q * shared, rows = n.tokens * shared;  // of a sequence, of a KV head
  const bool together = n.groups > 0 && shared <= kTogether;
  r.few_groups = rows <= kRowTile;
  // tiles of 128 rows where some context has them; wide heads leave no registers for them
  // (Of a group of small chunks the prefix gains by them what own tokens, in tiles of few rows, lose.
  // us with tiles of 64 and of 128: 8 sequences of 5 queries and up to 1,024 tokens behind 4 Ki, 160
  // rows, 41 and 55; of 16 queries, 512 rows, 49 and 59; 64 of 5 behind 8 Ki, 1,280 rows, 210 and 144.)
  const int64_t gains = most > kRowTile ? kWideGroup : kTogether;
  const bool wide = n.d <= 128 && (most > kTogether || (together && rows / n.groups > gains));
  r.row_tiles = wide ? 2 : 1;
  const int64_t tile = kRowTile * kFullWaves * r.row_tiles;
  const bool brief = n.groups == 0 && n.max_len <= kBrief;
  if (shared <= kRowTile)
    r.few = cut(n.seqs, n.heads, n.max_len, brief ? 1 : kFillRows, kRound, kEven, kEvenChunk);
  if (most > kRowTile)
    r.many = cut(least(n.seqs * ceil_div(most, tile),
                       rows / tile + least(n.seqs, rows / (kRowTile + 1))),
                 n.heads, n.max_len + n.max_prefix, kFillTiles, 2 * kRound, 0, 2 * kRound);
  // A prefix's parts are long ones where there is much to do beside them: 64 sequences of up to 1,024
  // tokens behind one prompt of 8 Ki 62 us for 65 (kFillTiles workgroups for it), 16 of 2,001 behind
  // 131 Ki, where they are all there is, 40 us for 48.
  const bool busy = static_cast<int64_t>(r.few.tiles) * r.few.splits * n.heads >= 2 * kFillTiles;
  if (together)
    r.group = r.few_groups ? cut(n.groups, n.heads, n.max_prefix, kFillRows, kRound, kEven, kEvenChunk)
                           : cut((rows + n.groups * (tile - 1)) / tile, n.heads, n.max_prefix,
                                 busy ? kFillTiles / 2 : kFillTiles, kRound, 0, kRound);
  // rows that are written where they go need no parts
  r.slots = r.group.splits + (r.many.splits > 1 || r.group.splits > 0 ? r.many.splits : 0);
  r.few_slots = r.few.splits > 1 || r.group.splits > 0 ? r.few.splits : 0;
  r.few_rows = least(most, kRowTile);
  const int64_t every = n.tokens * n.q_heads, few = n.seqs * n.heads * r.few_rows;
  if (n.mass && r.few.splits > 0) {
    r.stored = (n.max_len + 3) / 4 * 4;
    r.scores = r.stored <= kMostScores / 4 / few ? few * r.stored * 4 : 0;
    if (r.scores == 0) r.stored = 0;
  }
  const auto on16 = [](int64_t x) { return (x + 15) / 16 * 16; };
  r.sums = r.slots * every * n.d * 4;
  r.stats = on16(r.slots * every * 8);
  r.few_sums = r.few_slots * few * n.d * 4;
  r.few_stats = on16((r.stored > 0 ? r.few.splits : r.few_slots) * few * 8);
  r.top = n.mass ? on16(every * 4) : 0;
  r.bytes = r.sums + r.stats + r.few_sums + r.few_stats + r.top + r.scores;
  return r;
}

// Workgroups of the launch, as full_attend has them.
int64_t workgroups(const Deal& r, int64_t heads) {
  const auto in = [&](const Cut& c) { return (c.splits * heads + 7) / 8 * 8 * c.tiles; };
  return in(r.group) + in(r.few) + in(r.many);
}

// What a length may be at most where the caller does not say.
int64_t room(int64_t given, int64_t width, int64_t block_size) {
  const int64_t most = least(width * block_size, (int64_t{1} << 31) - 1);
  return given == 0 ? most : least(given, most);
}

// Whether some row of the queries, `row` bytes each, has a byte of the `size` at `out`.
bool rows_meet(const void* q, int64_t by_token, int64_t tokens, int64_t by_head, int64_t heads,
               int64_t row, const void* out, int64_t size) {
  typedef __int128 Wide;
  if (by_token < 0) {  // the last token first
    const Wide last = static_cast<Wide>(reinterpret_cast<intptr_t>(q)) +
                      static_cast<Wide>(by_token) * (tokens - 1);
    q = reinterpret_cast<const void*>(static_cast<intptr_t>(last));
    by_token = -by_token;
  }
  const Wide from = reinterpret_cast<intptr_t>(q), at = reinterpret_cast<intptr_t>(out);
  const Wide span = static_cast<Wide>(by_token) * (tokens - 1) + row;
  const Wide heads_span = static_cast<Wide>(by_head) * (heads - 1);
  if (from + (heads_span < 0 ? heads_span : 0) >= at + size ||
      from + (heads_span > 0 ? heads_span : 0) + span <= at)
    return false;
  for (int64_t h = 0; h < heads; h++) {
    // the first of the head's rows that ends behind out's start
    const Wide first = from + static_cast<Wide>(by_head) * h;
    const Wide short_of = at - first - row;
    Wide t = 0;
    if (short_of >= 0) t = by_token > 0 ? short_of / by_token + 1 : static_cast<Wide>(tokens);
    if (t < tokens && first + t * by_token < at + size) return true;
  }
  return false;
}

}  // namespace
}  // namespace evs

extern "C" int evs_attend_workspace(int64_t seqs, int64_t tokens, int64_t q_heads, int64_t heads,
                                    int64_t head_dim, int64_t max_q, int64_t max_len,
                                    int64_t groups, int64_t max_prefix, int mass, int64_t* bytes) {
  evs::clear_error();
  EVS_REQUIRE(bytes != nullptr, "evs_attend_workspace: null result");
  *bytes = 0;
  const evs::Counts n{seqs,   tokens, q_heads, heads,      head_dim,
                      max_q, max_len, groups,  max_prefix, mass != 0};
  EVS_REQUIRE(evs::good(n), "evs_attend_workspace: bad count");
  if (seqs > 0 && tokens > 0 && max_q > 0) *bytes = evs::deal(n).bytes;
  return EVS_OK;
}

extern "C" int evs_attend(const void* q, const int64_t* q_strides, int type, void* out, float* lse,
                          int64_t tokens, int64_t q_heads, const void* cache, int64_t num_blocks,
                          int64_t block_size, int64_t heads, int64_t head_dim,
                          const int64_t* strides, const int32_t* tables, int64_t table_stride,
                          int64_t width, const int32_t* lens, const int32_t* q_starts,
                          int64_t seqs, int64_t max_q, int64_t max_len,
                          const int32_t* prefix_tables, int64_t prefix_stride,
                          int64_t prefix_width, const int32_t* prefix_lens,
                          const int32_t* group_starts, int64_t groups, int64_t max_prefix,
                          float* mass, float scale, void* workspace, int64_t workspace_bytes,
                          void* stream) {
  evs::clear_error();
  const char* who = "evs_attend";
  constexpr int64_t most = int64_t{1} << 31;
  EVS_REQUIRE(type == EVS_BF16 || type == EVS_F16, "%s: type %d: bf16 or f16", who, type);
  EVS_REQUIRE(head_dim >= evs::kFullMinDim && head_dim <= evs::kFullMaxDim && head_dim % 8 == 0,
              "%s: head size %lld: a multiple of 8 from %d to %d", who,
              static_cast<long long>(head_dim), evs::kFullMinDim, evs::kFullMaxDim);
  EVS_REQUIRE(num_blocks >= 0 && num_blocks < most && block_size > 0 && block_size < most &&
                  heads > 0 && heads < (1 << 16),
              "%s: bad cache: %lld pages of %lld slots and %lld heads", who,
              static_cast<long long>(num_blocks), static_cast<long long>(block_size),
              static_cast<long long>(heads));
  EVS_REQUIRE(width >= 0 && width < most && prefix_width >= 0 && prefix_width < most,
              "%s: bad table width", who);
  // (a context of both is numbered in 32 bits)
  EVS_REQUIRE(prefix_width == 0 || (width + prefix_width) * block_size < most,
              "%s: tables with room for %lld tokens of prefixes and %lld behind them: 2^31 tokens are "
              "too many",
              who, static_cast<long long>(prefix_width * block_size),
              static_cast<long long>(width * block_size));
  evs::Counts n{seqs,   tokens, q_heads, heads, head_dim,
                max_q, 0,      groups,  0,     mass != nullptr};
  EVS_REQUIRE(max_len >= 0 && max_prefix >= 0, "%s: bad count", who);
  EVS_REQUIRE(evs::good(n), "%s: bad count (%lld query heads on %lld)", who,
              static_cast<long long>(q_heads), static_cast<long long>(heads));
  const float scale_log2 = scale * 1.4426950408889634f;  // log2(e)
  EVS_REQUIRE(scale_log2 > 0 && scale_log2 < INFINITY,
              "%s: the scale must be positive and finite", who);
  EVS_REQUIRE(strides != nullptr, "%s: a layout is five strides", who);
  EVS_REQUIRE(strides[4] == 1, "%s: a row's elements must be contiguous (element stride %lld)", who,
              static_cast<long long>(strides[4]));
  bool aligned = reinterpret_cast<uintptr_t>(cache) % 16 == 0;
  for (int i = 0; i < 4; i++) aligned = aligned && strides[i] % 8 == 0;
  EVS_REQUIRE(aligned, "%s: the cache's rows must start on 16 bytes", who);
  if (tokens == 0 || seqs == 0 || max_q == 0) return EVS_OK;
  EVS_REQUIRE(q_starts != nullptr || (tokens == seqs && max_q == 1),
              "%s: without query starts there is one query a sequence: %lld queries, %lld sequences",
              who, static_cast<long long>(tokens), static_cast<long long>(seqs));
  EVS_REQUIRE(q != nullptr && q_strides != nullptr && out != nullptr && lens != nullptr &&
                  (cache != nullptr || num_blocks == 0) && (tables != nullptr || width == 0) &&
                  (groups == 0 || (prefix_lens != nullptr && group_starts != nullptr &&
                                   (prefix_tables != nullptr || prefix_width == 0))),
              "%s: null argument", who);
  EVS_REQUIRE(reinterpret_cast<uintptr_t>(out) % 16 == 0, "%s: out must start on 16 bytes", who);
  EVS_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0 && q_strides[0] % 8 == 0 &&
                  q_strides[1] % 8 == 0,
              "%s: queries must start on 16 bytes", who);
  n.max_len = evs::room(max_len, width, block_size);
  n.max_prefix = evs::room(max_prefix, prefix_width, block_size);
  const evs::Deal deal = evs::deal(n);
  // (a launch has at most 2^32 - 1 threads along x)
  EVS_REQUIRE(tokens < most / 256 &&
                  evs::workgroups(deal, heads) < most / 256,
              "%s: too many tiles of query rows", who);
  // (workgroups that weigh: at least one a context and head, and 2^20 more)
  EVS_REQUIRE(mass == nullptr || (seqs + groups) * heads < most / 512,
              "%s: too many sequences and heads to weigh", who);
  EVS_REQUIRE(deal.bytes <= workspace_bytes &&
                  (deal.bytes == 0 || (workspace != nullptr &&
                                       reinterpret_cast<uintptr_t>(workspace) % 16 == 0)),
              "%s: a workspace of %lld bytes on 16, %lld needed", who,
              static_cast<long long>(workspace_bytes), static_cast<long long>(deal.bytes));
  EVS_REQUIRE(!evs::rows_meet(q, q_strides[0] * 2, tokens, q_strides[1] * 2, q_heads, head_dim * 2,
                              out, tokens * q_heads * head_dim * 2),
              "%s: out must not be the queries nor overlap them: all heads' parts read them", who);
  evs::FullArgs a{};
  a.base = static_cast<char*>(const_cast<void*>(cache));
  a.sb = strides[0] * 2;
  a.so = strides[1] * 2;
  a.sh = strides[2] * 2;
  a.skv = strides[3] * 2;
  a.num_blocks = static_cast<int32_t>(num_blocks);
  a.block_size = static_cast<int32_t>(block_size);
  a.div_bs = evs::FastDiv(static_cast<uint32_t>(block_size));
  a.heads = static_cast<int32_t>(heads);
  a.d = static_cast<int32_t>(head_dim);
  a.q = static_cast<const char*>(q);
  a.q_token = q_strides[0] * 2;
  a.q_head = q_strides[1] * 2;
  a.out = static_cast<char*>(out);
  a.lse = lse;
  a.starts = q_starts;
  a.seqs = static_cast<int32_t>(seqs);
  a.tokens = static_cast<int32_t>(tokens);
  a.max_q = static_cast<int32_t>(max_q < tokens ? max_q : tokens);
  a.q_heads = static_cast<int32_t>(q_heads);
  a.shared = evs::FastDiv(static_cast<uint32_t>(q_heads / heads));
  a.div_heads = evs::FastDiv(static_cast<uint32_t>(heads));
  a.scale_log2 = scale_log2;
  a.group = deal.group;
  a.few = deal.few;
  a.many = deal.many;
  a.few_groups = deal.few_groups;
  a.row_tiles = deal.row_tiles;
  a.own.tables = tables;
  a.own.stride = table_stride;
  a.own.width = static_cast<int32_t>(width);
  a.own.lens = lens;
  a.own.n = a.seqs;
  if (groups > 0) {
    a.pre.tables = prefix_tables;
    a.pre.stride = prefix_stride;
    a.pre.width = static_cast<int32_t>(prefix_width);
    a.pre.lens = prefix_lens;
    a.pre.n = static_cast<int32_t>(groups);
    a.group_starts = group_starts;
  }
  a.few_rows = static_cast<int32_t>(deal.few_rows);
  char* at = static_cast<char*>(workspace);
  const auto take = [&](int64_t bytes) {
    float* p = reinterpret_cast<float*>(at);
    at += bytes;
    return p;
  };
  a.parts.sums = take(deal.sums);
  a.parts.stats = take(deal.stats);
  a.few_parts.sums = take(deal.few_sums);
  a.few_parts.stats = take(deal.few_stats);
  if (mass != nullptr) {
    a.mass = mass;
    a.top = take(deal.top);
    if (deal.stored > 0) a.scores = take(deal.scores);
    a.stored = static_cast<int32_t>(deal.stored);
  }
  const hipStream_t s = evs::as_stream(stream);
  if (mass != nullptr && q_starts != nullptr && groups > 0) {
    // A prefix's tokens are weighed by all queries of its group (group_rows), whichever part took the
    // prefix: those that no sequence names, or that are past max_q, have no weights.
    const int64_t rows = tokens * q_heads;
    evs::no_weights<<<static_cast<uint32_t>((rows + 255) / 256), evs::kFullThreads, 0, s>>>(a.top,
                                                                                          rows);
    EVS_LAUNCHED(who);
  }
  if (const int rc = evs::full_attend(a, type, s)) return rc;
  // workgroups that join rows, enough of them for each query to fill the GPU, and that weigh tokens
  const int64_t slots = deal.group.splits + (deal.few.splits > deal.many.splits ? deal.few.splits
                                                                                : deal.many.splits);
  evs::JoinShape shape{};
  int64_t pieces = 1, down = 1;
  {
    // four elements a thread; a row in pieces of 32 elements where there are many parts of few rows
    while ((4 << shape.words) < head_dim) shape.words++;
    if (slots >= 32 && tokens * q_heads < 2048)
      while (shape.words > 3) shape.words--;
    pieces = (head_dim / 4 + (1 << shape.words) - 1) >> shape.words;
    while (shape.words + shape.turns < 8 && (8 << shape.turns) < slots) shape.turns++;
    const int64_t heads_at = evs::kFullThreads >> (shape.words + shape.turns);
    down = (q_heads + heads_at - 1) / heads_at * pieces;
    if (down > 4096 / tokens + 1) down = 4096 / tokens + 1;
  }
  shape.pieces = evs::FastDiv(static_cast<uint32_t>(pieces));
  shape.down = evs::FastDiv(static_cast<uint32_t>(down));
  const int64_t joins = deal.slots + deal.few_slots > 0 ? tokens * down : 0;
  const int64_t steps = deal.stored > 0 ? (deal.stored + evs::kScored - 1) / evs::kScored : 0;
  const int64_t items = joins + seqs * heads * steps;
  if (items > 0) {
    const evs::FastDiv by_steps(static_cast<uint32_t>(steps > 0 ? steps : 1));
    const uint32_t grid = static_cast<uint32_t>(items), first = static_cast<uint32_t>(joins);
    if (type == EVS_BF16)
      evs::join_full<__bf16><<<grid, evs::kFullThreads, 0, s>>>(a, first, shape, by_steps);
    else
      evs::join_full<_Float16><<<grid, evs::kFullThreads, 0, s>>>(a, first, shape, by_steps);
    EVS_LAUNCHED(who);
  }
  // what is left to weigh: prefixes, contexts of many rows, tokens without a score
  const bool left = deal.group.tiles > 0 || deal.many.tiles > 0 ||
                    deal.stored < evs::room(0, width, block_size);
  return mass == nullptr || !left ? EVS_OK
                                  : evs::full_weigh(a, type, n.max_len, n.max_prefix, s);
}
