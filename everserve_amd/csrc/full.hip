// Attention over full-width pages: the calls, how their work is dealt out, and the join of contexts
// in several parts (full.hpp has the mathematics, full_attend.hip and full_weigh.hip the
// kernels).
#include "full.hpp"

namespace evs {
namespace {

// Rows of one query joined from their parts: four elements a thread, and the parts in turn to as many
// threads as there may be parts for; the rest of a workgroup takes further heads. Bound by latency
// where parts are many, else by their bytes.
template <typename T>
__global__ __launch_bounds__(kFullThreads) void join_full(FullArgs a, int word_bits,
                                                          int turn_bits) {
  __shared__ f32x4 s_v[kFullThreads];
  __shared__ float s_m[kFullThreads], s_l[kFullThreads];
  const int token = blockIdx.x;
  const int s = sequence_of(a, token);
  if (s < 0) return;  // uniform
  const Rows sq = scalar_rows(sequence_rows(a, s));
  const int tid = threadIdx.x;
  const int w = tid & ((1 << word_bits) - 1);
  const int turn = (tid >> word_bits) & ((1 << turn_bits) - 1);
  const int heads_at = kFullThreads >> (word_bits + turn_bits);
  const int q_head = blockIdx.y * heads_at + (tid >> (word_bits + turn_bits));
  const int shared = a.shared.d;
  // the tokens that the row's tile sees, and its parts
  const bool few = sq.rows <= kRowTile, alone = sq.rows > kTogether;
  const int g = a.group.tiles > 0 || (alone && a.pre.n > 0) ? group_of(a, s) : -1;
  const int prefix = g < 0 ? 0 : length_of(a, a.pre, g);
  const int ahead = alone ? prefix : 0;
  const int in = min(q_head, a.q_heads - 1);
  const int row = (token - sq.q0) * shared + in % shared;
  const int tile = few ? kRowTile : kRowTile * kFullWaves * a.row_tiles;
  const int last = min(row / tile * tile + tile, sq.rows) - 1;
  const int end = min(ahead + sq.len, max(ahead + sq.len - sq.nq + last / shared + 1, ahead));
  const Cut& cut = few ? a.few : a.many;
  const bool joined = q_head < a.q_heads && is_joined(a, cut, sq.rows, end);
  const int before = alone || !joined ? 0 : parts_of(a.group, prefix);
  const int parts = joined ? before + max(parts_of(cut, end), 1) : 0;
  float top = -INFINITY, total = 0;
  f32x4 v = {0, 0, 0, 0};
  const int wr = min(w, a.d / 4 - 1);
#pragma unroll 4
  for (int k = turn; k < parts; k += 1 << turn_bits) {
    const int slot = k < before ? k : a.group.splits + k - before;
    const int64_t at = part_at(a, slot, token, in);
    const float m = a.stats[2 * at], l = a.stats[2 * at + 1];
    const f32x4 y = *reinterpret_cast<const f32x4*>(a.sums + at * a.d + 4 * wr);
    const float now = fmaxf(top, m);
    const float ref = now == -INFINITY ? 0.0f : now;
    const float f = __builtin_amdgcn_exp2f(top - ref), h = __builtin_amdgcn_exp2f(m - ref);
    top = now;
    total = total * f + l * h;
    v = v * f + y * h;
  }
  if (turn_bits > 0) {
    s_v[tid] = v;
    s_m[tid] = top;
    s_l[tid] = total;
    __syncthreads();
    if (turn != 0) return;
    for (int k = 1; k < 1 << turn_bits; k++) top = fmaxf(top, s_m[tid + (k << word_bits)]);
    const float ref = top == -INFINITY ? 0.0f : top;
    total = 0;
    v = f32x4{0, 0, 0, 0};
    for (int k = 0; k < 1 << turn_bits; k++) {
      const int t = tid + (k << word_bits);
      const float f = __builtin_amdgcn_exp2f(s_m[t] - ref);
      total += s_l[t] * f;
      v += s_v[t] * f;
    }
  }
  if (joined && w < a.d / 4) finish4<T>(a, token, q_head, w, v, top, total);
}

__global__ __launch_bounds__(kFullThreads) void no_weights(float* top, int64_t n) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kFullThreads + threadIdx.x;
  if (i < n) top[i] = INFINITY;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t least(int64_t a, int64_t b) { return a < b ? a : b; }

constexpr int64_t kRound = 256;  // tokens that a workgroup's waves take in turn, of few rows
constexpr int64_t kFillRows = 1024;  // workgroups that fill the GPU, of few rows
constexpr int64_t kFillTiles = 256;  // and of many
constexpr int64_t kMostParts = 64;

// How contexts of up to max_len tokens are cut for `tiles` row tiles that there may be: into parts
// that make `fill` workgroups in all, of `least_chunk` tokens at least.
Cut cut(int64_t tiles, int64_t heads, int64_t max_len, int64_t fill, int64_t least_chunk) {
  Cut c{};
  if (tiles == 0) return c;
  int64_t parts = least(least(ceil_div(fill, tiles * heads), kMostParts),
                        ceil_div(max_len, least_chunk));
  parts = parts < 1 ? 1 : parts;
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
  int64_t slots, sums, stats, top, bytes;
};

Deal deal(Counts n) {
  Deal r{};
  const int64_t shared = n.q_heads / n.heads;
  if (n.max_q > n.tokens) n.max_q = n.tokens;
  const int64_t most = n.max_q * shared, rows = n.tokens * shared;  // of a sequence, of a KV head
  const bool together = n.groups > 0 && shared <= kTogether;
  r.few_groups = rows <= kRowTile;
  // tiles of 128 rows where some context has them; wide heads leave no registers for them
  const bool wide = n.d <= 128 && (most > kTogether || (together && rows / n.groups > kTogether));
  r.row_tiles = wide ? 2 : 1;
  const int64_t tile = kRowTile * kFullWaves * r.row_tiles;
  if (shared <= kRowTile) r.few = cut(n.seqs, n.heads, n.max_len, kFillRows, kRound);
  if (most > kRowTile)
    r.many = cut(least(n.seqs * ceil_div(most, tile),
                       rows / tile + least(n.seqs, rows / (kRowTile + 1))),
                 n.heads, n.max_len + n.max_prefix, kFillTiles, 2 * kRound);
  if (together)
    r.group = r.few_groups ? cut(n.groups, n.heads, n.max_prefix, kFillRows, kRound)
                           : cut(rows / tile + n.groups, n.heads, n.max_prefix, kFillTiles, kRound);
  r.slots = r.group.splits + (r.few.splits > r.many.splits ? r.few.splits : r.many.splits);
  if (r.slots == 1) r.slots = 0;
  const int64_t every = n.tokens * n.q_heads;
  r.sums = r.slots * every * n.d * 4;
  r.stats = r.slots * every * 8;
  r.top = n.mass ? every * 4 : 0;
  r.bytes = (r.sums + r.stats + r.top + 15) / 16 * 16;
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
  evs::Counts n{seqs,   tokens, q_heads, heads, head_dim,
                max_q, 0,      groups,  0,     mass != nullptr};
  EVS_REQUIRE(max_len >= 0 && max_prefix >= 0, "%s: bad count", who);
  EVS_REQUIRE(evs::good(n), "%s: bad count (%lld query heads on %lld)", who,
              static_cast<long long>(q_heads), static_cast<long long>(heads));
  EVS_REQUIRE(scale > 0 && scale < INFINITY, "%s: the scale must be positive and finite", who);
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
  EVS_REQUIRE(deal.bytes <= workspace_bytes &&
                  (deal.bytes == 0 || (workspace != nullptr &&
                                       reinterpret_cast<uintptr_t>(workspace) % 16 == 0)),
              "%s: a workspace of %lld bytes on 16, %lld needed", who,
              static_cast<long long>(workspace_bytes), static_cast<long long>(deal.bytes));
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
  a.scale_log2 = scale * 1.4426950408889634f;
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
  char* at = static_cast<char*>(workspace);
  a.sums = reinterpret_cast<float*>(at);
  a.stats = reinterpret_cast<float*>(at + deal.sums);
  if (mass != nullptr) {
    a.mass = mass;
    a.top = reinterpret_cast<float*>(at + deal.sums + deal.stats);
  }
  const hipStream_t s = evs::as_stream(stream);
  if (mass != nullptr && q_starts != nullptr) {
    // queries that no sequence names have no weights
    const int64_t rows = tokens * q_heads;
    evs::no_weights<<<static_cast<uint32_t>((rows + 255) / 256), evs::kFullThreads, 0, s>>>(a.top,
                                                                                          rows);
    EVS_LAUNCHED(who);
  }
  if (const int rc = evs::full_attend(a, type, s)) return rc;
  if (deal.slots > 0) {
    int word_bits = 0, turn_bits = 0;
    while ((4 << word_bits) < head_dim) word_bits++;
    while (word_bits + turn_bits < 8 && (4 << turn_bits) < deal.slots) turn_bits++;
    const int64_t heads_at = evs::kFullThreads >> (word_bits + turn_bits);
    const dim3 grid(static_cast<uint32_t>(tokens),
                    static_cast<uint32_t>((q_heads + heads_at - 1) / heads_at));
    if (type == EVS_BF16)
      evs::join_full<__bf16><<<grid, evs::kFullThreads, 0, s>>>(a, word_bits, turn_bits);
    else
      evs::join_full<_Float16><<<grid, evs::kFullThreads, 0, s>>>(a, word_bits, turn_bits);
    EVS_LAUNCHED(who);
  }
  return mass == nullptr ? EVS_OK : evs::full_weigh(a, type, n.max_len, n.max_prefix, s);
}
