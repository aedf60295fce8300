// The weights that tokens got in an attention over full-width pages, added to their mass.
//
// The weight of token t for row r is exp(s_rt - lse_r), with the row's lse from the attention before
// it; a token's mass of a KV head grows by their sum over the rows of that head that see it. The sum
// is formed by the wave that has the token, row tile by row tile; from 64 rows on by the four waves of
// a workgroup, which share the rows and join their sums in LDS; or, of few rows' own tokens, by a
// thread from the scores that the attention kept (weigh_scores in full.hip). Each in a fixed order,
// without atomics: the same sums in every run. A prefix's tokens get the weights of all rows of its
// group at once.
#include "full.hpp"

namespace evs {
namespace {

// Tokens of a wave, whose keys stay in registers while the rows pass.
template <int NG>
constexpr int kKept = NG > 4 ? 32 : 64;
// Rows from which a workgroup's waves share them, not the tokens: each then has a tile of them.
constexpr int kManyRows = 64;

// One workgroup: the tokens of a context and KV head from kKept times `at` on, at every so-many-th
// place. The rows of a context with many are dealt to the waves in tiles of 16, and a token's sums
// joined in LDS; else each wave has tokens of its own.
//
// Where rows are many, K stays in registers and the queries pass through LDS, so the kernel is bound by
// its vector arithmetic: for 16 rows of 64 tokens of 128 elements some 130 instructions, 16
// exponentials, multiply-adds and adds among them, beside 16 matrix instructions. Two chunks of 1,024
// queries that end at up to 4,001 tokens, behind 1,000 (32 heads of 128 on 8): 99 us of the call's 288,
// which took 310 with queries read as operands. Where rows are few it is bound by reading K; of few
// rows' own tokens the attention's scores are read instead (full.hip): a decode step of 64 sequences
// of 1 to 4 Ki 185 us for 243.
template <typename T, int NG>
__global__ __launch_bounds__(kFullThreads) void weigh_full(FullArgs a, uint32_t prefix_items,
                                                           FastDiv prefix_steps, FastDiv own_steps) {
  constexpr int kG = kKept<NG> / 16;
  __shared__ float s_sum[kFullWaves][kKept<NG>];
  // a wave's queries, as full_tiles.hpp keeps keys
  __shared__ u32x4 s_query[kFullWaves][NG][64];
  const bool prefix = blockIdx.x < prefix_items;
  const Contexts& c = prefix ? a.pre : a.own;
  const FastDiv& steps = prefix ? prefix_steps : own_steps;
  uint32_t head, rest, who, at;
  a.div_heads.divmod(prefix ? blockIdx.x : blockIdx.x - prefix_items, rest, head);
  steps.divmod(rest, who, at);
  const Rows sq = scalar_rows(prefix ? group_rows(a, who) : sequence_rows(a, who));
  if (sq.rows == 0) return;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int past = prefix ? sq.len : sq.len - sq.nq;
  const int32_t* table = c.tables + static_cast<int64_t>(who) * c.stride;
  const uint64_t base = reinterpret_cast<uint64_t>(a.base) + head * a.sh;
  const bool by_rows = sq.rows >= kManyRows;
  const int64_t span = by_rows ? kKept<NG> : kKept<NG> * kFullWaves;
  const int row_step = by_rows ? kRowTile * kFullWaves : kRowTile;
  // tokens that the scores kept have been weighed by
  const int64_t done = !prefix && sq.rows <= kRowTile ? a.stored : 0;
  for (int64_t first = done + at * span + (by_rows ? 0 : kKept<NG> * wave); first < sq.len;
       first += steps.d * span) {
    const int t = static_cast<int>(first);
    u32x4 k[kG][NG];
#pragma unroll
    for (int g = 0; g < kG; g++) {
      uint32_t n, off;
      a.div_bs.divmod(min(static_cast<uint32_t>(t) + 16 * g + col,
                          static_cast<uint32_t>(sq.len) - 1),
                      n, off);
      const int32_t page = table[n];
      const bool ok = page >= 0 && page < a.num_blocks;
      const uint64_t p = base + (ok ? page * a.sb + static_cast<int64_t>(off) * a.so : 0);
#pragma unroll
      for (int i = 0; i < NG; i++) {
        const int e = 4 * i + quad;
        const bool in = 8 * e < a.d;
        const u32x4 x = load16(p + (in ? 16 * e : 0));
#pragma unroll
        for (int j = 0; j < 4; j++) k[g][i][j] = in ? x[j] : 0;
      }
    }
    float sum[kG][4];
#pragma unroll
    for (int g = 0; g < kG; g++)
#pragma unroll
      for (int r = 0; r < 4; r++) sum[g][r] = 0;
    const int from = max(t - past, 0) * static_cast<int>(a.shared.d);  // the first row that sees t
    const int row_first = from / kRowTile * kRowTile + (by_rows ? kRowTile * wave : 0);
    // The next tiles' queries are on their way, read row by row (as operands, 16 bytes of 16 rows side
    // by side, they took the memory pipeline four times as long).
    struct Tile {
      u32x4 x[NG];
      float top;
      int sees;  // the token of this lane's first that its row sees last
    };
    const auto load = [&](int row0, Tile& to) {
      uint32_t qi, qg;
      a.shared.divmod(min(row0 + col, sq.rows - 1), qi, qg);
      const int64_t token = sq.q0 + qi;
      const int q_head = head * a.shared.d + qg;
      const uint64_t p = reinterpret_cast<uint64_t>(a.q) + token * a.q_token + q_head * a.q_head;
#pragma unroll
      for (int n = 0; n < NG; n++) {
        const int row = (64 * n + lane) / (4 * NG), chunk = (64 * n + lane) % (4 * NG);
        const uint32_t lo = __shfl(static_cast<uint32_t>(p), row);
        const uint32_t hi = __shfl(static_cast<uint32_t>(p >> 32), row);
        const bool in = 8 * chunk < a.d;
        const u32x4 x = load16((static_cast<uint64_t>(hi) << 32 | lo) + (in ? 16 * chunk : 0));
#pragma unroll
        for (int j = 0; j < 4; j++) to.x[n][j] = in ? x[j] : 0;
      }
      to.top = row0 + col < sq.rows ? a.top[token * a.q_heads + q_head] : INFINITY;
      to.sees = past + static_cast<int>(qi) - t - 4 * quad;
    };
    constexpr int kTilesAhead = 2;
    Tile tiles[kTilesAhead];
#pragma unroll
    for (int n = 0; n < kTilesAhead; n++) load(row_first + n * row_step, tiles[n]);
    for (int row0 = row_first; row0 < sq.rows; row0 += kTilesAhead * row_step) {
#pragma unroll
      for (int n = 0; n < kTilesAhead; n++) {
        if (row0 + n * row_step >= sq.rows) break;
        Tile& x = tiles[n];
        wave_sync();  // the tile before has been read
#pragma unroll
        for (int i = 0; i < NG; i++) {
          const int row = (64 * i + lane) / (4 * NG), chunk = (64 * i + lane) % (4 * NG);
          s_query[wave][chunk >> 2][16 * (chunk & 3) + (row ^ (chunk & 15))] = x.x[i];
        }
        wave_sync();
        u32x4 q[NG];
#pragma unroll
        for (int i = 0; i < NG; i++) q[i] = s_query[wave][i][lane ^ ((4 * i + quad) & 15)];
        f32x4 acc[kG];
#pragma unroll
        for (int g = 0; g < kG; g++) acc[g] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < NG; i++)
#pragma unroll
          for (int g = 0; g < kG; g++) acc[g] = mma<T>(k[g][i], q[i], acc[g]);
        const float top = x.top;
        const int sees = x.sees;
        load(row0 + (n + kTilesAhead) * row_step, x);
        // (rows that see nothing have no weights, whatever their scores)
        const bool all = sees + 4 * quad >= kKept<NG> - 1 && top != INFINITY;
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(!all) != 0, false)) {
          asm volatile("");  // a branch: most rows see all of the tokens
#pragma unroll
          for (int g = 0; g < kG; g++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
              const float w =
                  __builtin_amdgcn_exp2f(__builtin_fmaf(acc[g][r], a.scale_log2, -top));
              sum[g][r] += sees >= 16 * g + r && top != INFINITY ? w : 0.0f;
            }
        } else {
#pragma unroll
          for (int g = 0; g < kG; g++)
#pragma unroll
            for (int r = 0; r < 4; r++)
              sum[g][r] += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[g][r], a.scale_log2, -top));
        }
      }
    }
    // over the rows of a tile, which are the lanes of a quarter
#pragma unroll
    for (int g = 0; g < kG; g++)
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) sum[g][r] += __shfl_xor(sum[g][r], d);
    // the sums before have been read
    if (by_rows)
      __syncthreads();
    else
      wave_sync();
    if (col == 0) {
#pragma unroll
      for (int g = 0; g < kG; g++)
#pragma unroll
        for (int r = 0; r < 4; r++) s_sum[wave][16 * g + 4 * quad + r] = sum[g][r];
    }
    if (by_rows)
      __syncthreads();
    else
      wave_sync();
    if (lane < kKept<NG> && (!by_rows || wave == 0)) {
      const uint32_t own = static_cast<uint32_t>(t) + lane;
      if (own < static_cast<uint32_t>(sq.len)) {
        float mine = s_sum[wave][lane];
        if (by_rows)
          for (int w = 1; w < kFullWaves; w++) mine += s_sum[w][lane];
        uint32_t n, off;
        a.div_bs.divmod(own, n, off);
        const int32_t page = table[n];
        if (page >= 0 && page < a.num_blocks) {
          float* m = a.mass + (static_cast<int64_t>(page) * a.heads + head) * a.block_size + off;
          *m = (!prefix && static_cast<int>(own) >= past ? 0.0f : *m) + mine;
        }
      }
    }
  }
}

template <typename T>
void launch(const FullArgs& a, uint32_t items, uint32_t prefix_items, FastDiv prefix_steps,
            FastDiv own_steps, hipStream_t s) {
  const int g = (a.d + 31) / 32;
  if (g <= 2)
    weigh_full<T, 2><<<items, kFullThreads, 0, s>>>(a, prefix_items, prefix_steps, own_steps);
  else if (g <= 3)
    weigh_full<T, 3><<<items, kFullThreads, 0, s>>>(a, prefix_items, prefix_steps, own_steps);
  else if (g <= 4)
    weigh_full<T, 4><<<items, kFullThreads, 0, s>>>(a, prefix_items, prefix_steps, own_steps);
  else if (g <= 6)
    weigh_full<T, 6><<<items, kFullThreads, 0, s>>>(a, prefix_items, prefix_steps, own_steps);
  else
    weigh_full<T, 8><<<items, kFullThreads, 0, s>>>(a, prefix_items, prefix_steps, own_steps);
}

// Workgroups that take the places of a context in turn: one a place, fewer where there are very many.
uint32_t steps_of(const FullArgs& a, int64_t max_len, int64_t contexts, int64_t rows) {
  const int64_t kept = (a.d > 128 ? 32 : 64) * (rows >= kManyRows ? 1 : kFullWaves);
  const int64_t steps = (max_len + kept - 1) / kept;
  const int64_t most = (int64_t{1} << 20) / (contexts * a.heads) + 1;
  const int64_t n = steps < most ? steps : most;
  return static_cast<uint32_t>(n < 1 ? 1 : n);
}

}  // namespace

int full_weigh(const FullArgs& a, int type, int64_t max_len, int64_t max_prefix, hipStream_t s) {
  const int64_t shared = a.shared.d, most = a.max_q * shared;  // rows of a sequence
  // (where the scores of few rows are kept only tokens past them are left, which there rarely are)
  const bool mostly = a.stored > 0 && most <= kRowTile;
  const FastDiv own(mostly ? 1 : steps_of(a, max_len, a.own.n, most));
  const FastDiv pre(a.pre.n > 0 ? steps_of(a, max_prefix, a.pre.n, a.tokens * shared) : 1);
  const int64_t prefix_items = static_cast<int64_t>(a.pre.n) * pre.d * a.heads;
  const int64_t items = prefix_items + static_cast<int64_t>(a.own.n) * own.d * a.heads;
  if (type == EVS_BF16)
    launch<__bf16>(a, static_cast<uint32_t>(items), static_cast<uint32_t>(prefix_items), pre, own,
                   s);
  else
    launch<_Float16>(a, static_cast<uint32_t>(items), static_cast<uint32_t>(prefix_items), pre, own,
                     s);
  EVS_LAUNCHED("evs_attend");
  return EVS_OK;
}

}  // namespace evs
