// Attention over a paged cache held in 4 bits: the calls, how their work is dealt out, and the join
// of contexts that were split (attend.hpp has the mathematics, attend_few.hip and attend_many.hip
// the kernels).
#include "attend.hpp"

namespace evs {
namespace {

constexpr int kJoinThreads = 256;

// Rows of a row tile that was split, joined: workgroups for each row tile that there may be and
// head, which take the tile's rows in turn. A workgroup's threads are dealt a dword of elements
// each and, as many times over as there are parts for, the parts in turn; the rest of them takes
// further rows.
//
// A launch of its own. After attend_few it is bound by latency: 4 to 7 us, a decode step of 64
// sequences 4.8. After attend_many it is bound by the parts' bytes: up to two a workgroup of 128
// rows, 68 MB for heads of 128, in 14 to 19 us. Joined by the last of a tile's workgroups to end
// instead, a decode step that took 86 us then took 113 with parts that pass the caches, and 417
// with fences of the GPU's scope.
template <bool kMany, typename T>
__global__ __launch_bounds__(kJoinThreads) void join_parts(AttendArgs a) {
  __shared__ float s_v[kJoinThreads][8 + 1];
  __shared__ float s_m[kJoinThreads];
  __shared__ float s_l[kJoinThreads];
  const Dealt& dealt = kMany ? a.many : a.few;
  uint32_t head, at, seq, tile;
  a.heads.divmod(blockIdx.x, at, head);
  const uint4 in = dealt.tiles_in[at];
  uint32_t owner, parts;
  if (kMany) {
    if (in.z < 2) return;
    seq = __builtin_amdgcn_readfirstlane(in.x);
    tile = __builtin_amdgcn_readfirstlane(in.y);
    owner = at;
    parts = __builtin_amdgcn_readfirstlane(in.z);
  } else {
    dealt.most.divmod(at, seq, tile);
    owner = __builtin_amdgcn_readfirstlane(in.x);
    parts = __builtin_amdgcn_readfirstlane(in.y);
  }
  const Sequence sq = sequence_of_all(a, seq);
  if (!kMany && (tile >= tiles_of<kMany>(a, sq) || parts == 1)) return;  // no tile: `in` is garbage
  // threads: [row][turn][dword], a row's dwords rounded up to a power of two
  const uint32_t lanes = 1u << a.join_bits;
  uint32_t turn_bits = 0;
  while ((lanes << turn_bits) < kJoinThreads && (2u << turn_bits) < parts) turn_bits++;
  const uint32_t turns = 1u << turn_bits;
  const uint32_t rows = kJoinThreads >> (a.join_bits + turn_bits);  // at once
  const uint32_t w = threadIdx.x & (lanes - 1), turn = (threadIdx.x >> a.join_bits) & (turns - 1);
  const uint32_t mine = threadIdx.x >> (a.join_bits + turn_bits);
  const uint32_t wr = min(w, static_cast<uint32_t>(a.c.W) - 1);
  const int row0 = static_cast<int>(tile << dealt.tile_bits);
  const uint32_t held = min(1 << dealt.tile_bits, sq.rows - row0);  // rows of it
  for (uint32_t r0 = blockIdx.y * rows; r0 < held; r0 += gridDim.y * rows) {
    const uint32_t r = r0 + mine;
    const int row = static_cast<int>(min(r, held - 1));
    float top = -INFINITY, total = 0, v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 4
    for (uint32_t k = turn; k < parts; k += turns) {
      const float* p = part_row(a, dealt, owner + k, k == 0, head, row);
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
    __syncthreads();  // the rows before have been read
    s_m[threadIdx.x] = top;
    s_l[threadIdx.x] = total;
#pragma unroll
    for (int j = 0; j < 8; j++) s_v[threadIdx.x][j] = v[j];
    __syncthreads();
    if (turn != 0 || w >= static_cast<uint32_t>(a.c.W) || r >= held) continue;
    for (uint32_t k = 1; k < turns; k++) top = fmaxf(top, s_m[threadIdx.x + (k << a.join_bits)]);
    const float ref = top == -INFINITY ? 0.0f : top;
    total = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = 0;
    for (uint32_t k = 0; k < turns; k++) {
      const uint32_t t = threadIdx.x + (k << a.join_bits);
      const float f = __builtin_amdgcn_exp2f(s_m[t] - ref);
      total += s_l[t] * f;
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] += s_v[t][j] * f;
    }
    finish<T>(a, sq, row0 + static_cast<int>(r), head, w, v, top, total);
  }
}

template <bool kMany>
int join(const AttendArgs& a, int type, hipStream_t s) {
  const Dealt& dealt = kMany ? a.many : a.few;
  const uint32_t rows = static_cast<uint32_t>(dealt.rows);
  const uint32_t heads = static_cast<uint32_t>(a.c.heads);
  const uint32_t across =
      (kMany ? dealt.workgroups : static_cast<uint32_t>(a.seqs) * dealt.most.d) * heads;
  // a workgroup a row where there are few tiles
  uint32_t down = (kMany ? 4096 : 1024) / across;
  down = down < 1 ? 1 : down > rows ? rows : down;
  const dim3 grid(across, down);
  if (type == EVS_BF16)
    join_parts<kMany, __bf16><<<grid, kJoinThreads, 0, s>>>(a);
  else
    join_parts<kMany, _Float16><<<grid, kJoinThreads, 0, s>>>(a);
  EVS_LAUNCHED("evs_fp4_attend");
  return EVS_OK;
}

// Workgroups of a kernel that the GPU holds at once: shares are made for so many, to end together.
constexpr int64_t kCus = 256;
int64_t few_at_once(int64_t d) { return (d > 64 ? 1 : 2) * kCus; }
constexpr int64_t kManyAtOnce = 2 * kCus;

constexpr int64_t kFewRows[] = {64, 128};
constexpr int64_t kLittle = 1 << 18;  // tokens of all sequences and KV heads

// How a call's work is dealt out, from its counts alone (the lengths are on the device).
struct Deal {
  Dealt few, many;
  uint32_t held;  // KV heads that a workgroup of attend_few takes
  int64_t few_rows;
  int64_t few_bytes, many_bytes;  // of the parts' workspace
};

// `tiles`: row tiles that there may be, `most` of one sequence; `in`: entries of tiles_in (0: one a
// workgroup); `groups`: workgroups that share a place in the line.
void deal_tiles(Dealt& r, int64_t& bytes, int64_t tiles, int64_t most, int64_t in, int64_t rows,
                int64_t groups, int64_t heads, int64_t d, int64_t max_len, int64_t at_once) {
  // (more sequences and heads than 2^24 leave no context to split)
  r.split = tiles * groups < 4 * at_once && max_len > 2 * kMinShare &&
            in * heads < (int64_t{1} << 24);
  int64_t workgroups = r.split ? at_once / groups : tiles;
  workgroups = workgroups < 1 ? 1 : workgroups;
  workgroups = (workgroups + 7) / 8 * 8;
  const int64_t bound = int64_t{1} << 30;  // more are refused by the caller
  r.workgroups = static_cast<uint32_t>(workgroups < bound ? workgroups : bound);
  r.rows = static_cast<int32_t>(rows);
  if (r.split) {
    r.most = FastDiv(static_cast<uint32_t>(most));
    r.in = in > 0 ? in : workgroups;
    bytes = r.in * 16 + (workgroups * 2 * heads * rows * (d + 2) * 4 + 15) / 16 * 16;
  }
}

void place_parts(Dealt& r, void* at) {
  r.tiles_in = static_cast<uint4*>(at);
  r.part = reinterpret_cast<float*>(static_cast<char*>(at) + r.in * 16);
}

// The most query rows a KV head of a sequence that attend_few takes. Up to 64, it wins throughout
// (32 heads on 8 of 128, us, it for attend_many: 4 sequences of 4 to 8 Ki tokens 50 for 70; 64 of 1
// to 2 Ki with 48 rows 87 for 131, with 64 level). From there to 128 it wins while there is little
// to do, where tiles of 128 rows leave most CUs idle: 4 sequences of 4 to 8 Ki with 128 rows 63 for
// 80, 16 of 1 to 2 Ki 65 for 78; but 24 of them 86 for 81, 32 107 for 85, 16 of 4 to 8 Ki 173 for
// 115.
int64_t few_rows(int64_t seqs, int64_t heads, int64_t max_len) {
  return max_len > 0 && seqs * heads > kLittle / max_len ? kFewRows[0] : kFewRows[1];
}

Deal deal(int64_t seqs, int64_t tokens, int64_t shared, int64_t heads, int64_t d, int64_t max_q,
          int64_t max_len, int64_t few_rows, bool side_by_side) {
  Deal r{};
  const auto least = [](int64_t x, int64_t y) { return x < y ? x : y; };
  const int64_t rows = max_q * shared;
  r.few_rows = few_rows;
  // row tiles: a sequence's rows, rounded up
  if (shared <= r.few_rows) {
    const int64_t most = (least(rows, r.few_rows) + kFewTile - 1) / kFewTile;
    const int64_t tiles = least(most * seqs, tokens * shared / kFewTile + seqs);
    // The most heads, up to the waves, that leave shares for all workgroups: heads that lie side by
    // side share memory lines (8 of 128: 5.4 TB/s, in fours 4.4 and in twos 3.2), but the more of
    // them a workgroup has, the fewer tokens its waves take at once.
    const int64_t shares = tiles * least(max_len / kMinShare + 1, few_at_once(d));
    r.held = 1;
    for (int64_t n = 2; side_by_side && n <= kFewWaves; n++)
      if (heads % n == 0 && shares * (heads / n) >= few_at_once(d))
        r.held = static_cast<uint32_t>(n);
    r.few.tile_bits = 4;
    deal_tiles(r.few, r.few_bytes, tiles, most, most * seqs, least(rows, kFewTile),
               heads / r.held, heads, d, max_len, few_at_once(d));
  }
  if (rows > r.few_rows) {
    const int64_t tile = many_tile(d);
    const int64_t most = (rows + tile - 1) / tile;
    const int64_t tiles = least(most * seqs, tokens * shared / tile + seqs);
    r.many.tile_bits = tile == 64 ? 6 : 7;
    deal_tiles(r.many, r.many_bytes, tiles, most, 0, least(rows, tile), heads, heads, d, max_len,
               kManyAtOnce);
  }
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
  // (the call takes max_len up to the tables' room: less may change who takes which rows)
  for (const int64_t few_rows : evs::kFewRows)
    for (const bool side_by_side : {false, true}) {
      const evs::Deal deal =
          evs::deal(seqs, tokens, q_heads / heads, heads, head_dim,
                    max_q < tokens ? max_q : tokens, max_len, few_rows, side_by_side);
      const int64_t need = deal.few_bytes + deal.many_bytes;
      if (need > *bytes) *bytes = need;
    }
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
  // a workgroup takes several heads where a token's rows of them follow one another
  const bool side_by_side = strides[2] > 0 && strides[2] <= 2 * evs::fp4_row_bytes(head_dim);
  const evs::Deal deal =
      evs::deal(seqs, tokens, shared, heads, head_dim, max_q, max_len,
                evs::few_rows(seqs, heads, max_len), side_by_side);
  const int64_t tiles =
      (static_cast<int64_t>(deal.few.workgroups) + deal.many.workgroups) * heads;
  EVS_REQUIRE(tiles < (int64_t{1} << 24), "%s: %lld tiles of query rows: below 2^24", who,
              static_cast<long long>(tiles));
  const int64_t need = deal.few_bytes + deal.many_bytes;
  EVS_REQUIRE(need <= workspace_bytes &&
                  (need == 0 || (workspace != nullptr &&
                                 reinterpret_cast<uintptr_t>(workspace) % 16 == 0)),
              "%s: a workspace of %lld bytes on 16, %lld needed", who,
              static_cast<long long>(workspace_bytes), static_cast<long long>(need));
  a.few_rows = static_cast<int32_t>(deal.few_rows);
  a.few = deal.few;
  a.many = deal.many;
  if (need > 0) {
    evs::place_parts(a.few, workspace);
    evs::place_parts(a.many, static_cast<char*>(workspace) + deal.few_bytes);
  }
  const uint32_t held = deal.held > 0 ? deal.held : 1;
  a.held = evs::FastDiv(held);
  a.turns = evs::kFewWaves / held;
  a.groups = evs::FastDiv(static_cast<uint32_t>(heads) / held);
  while ((1 << a.join_bits) < a.c.W) a.join_bits++;
  const hipStream_t s = evs::as_stream(stream);
  if (a.few.workgroups > 0) {
    if (const int rc = evs::attend_few(a, type, s)) return rc;
    if (a.few.split)
      if (const int rc = evs::join<false>(a, type, s)) return rc;
  }
  if (a.many.workgroups > 0) {
    if (const int rc = evs::attend_many(a, type, s)) return rc;
    if (a.many.split)
      if (const int rc = evs::join<true>(a, type, s)) return rc;
  }
  return EVS_OK;
}
