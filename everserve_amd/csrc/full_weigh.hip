// The weights that tokens got in an attention over full-width pages, added to their mass.
//
// The weight of token t for row r is exp(s_rt - lse_r), with the row's lse from the attention before
// it; a token's mass of a KV head grows by their sum over the rows of that head that see it. Each
// token and head has one wave, which takes the rows in order: no atomics, and the same sums in every
// run. A prefix's tokens get the weights of all rows of its group at once.
#include "full.hpp"

namespace evs {
namespace {

constexpr int kStep = 32 * kFullWaves;  // tokens of a workgroup

// One workgroup: every so-many-th 128 tokens of a context and KV head, 32 of them a wave, whose keys
// stay in registers while the rows pass.
template <typename T, int NG>
__global__ __launch_bounds__(kFullThreads) void weigh_full(FullArgs a, uint32_t prefix_items,
                                                           FastDiv prefix_steps, FastDiv own_steps) {
  const bool prefix = blockIdx.x < prefix_items;
  const Contexts& c = prefix ? a.pre : a.own;
  const FastDiv& steps = prefix ? prefix_steps : own_steps;
  uint32_t head, rest, who, at;
  a.div_heads.divmod(prefix ? blockIdx.x : blockIdx.x - prefix_items, rest, head);
  steps.divmod(rest, who, at);
  const Rows sq = scalar_rows(prefix ? group_rows(a, who) : sequence_rows(a, who));
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int past = prefix ? sq.len : sq.len - sq.nq;
  const int32_t* table = c.tables + static_cast<int64_t>(who) * c.stride;
  const uint64_t base = reinterpret_cast<uint64_t>(a.base) + head * a.sh;
  for (int64_t first = static_cast<int64_t>(at) * kStep + 32 * wave; first < sq.len;
       first += static_cast<int64_t>(steps.d) * kStep) {
    const int t = static_cast<int>(first);
    u32x4 k[2][NG];
#pragma unroll
    for (int g = 0; g < 2; g++) {
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
    float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    const int from = max(t - past, 0) * static_cast<int>(a.shared.d);  // the first row that sees t
    for (int row0 = from / kRowTile * kRowTile; row0 < sq.rows; row0 += kRowTile) {
      const bool in = row0 + col < sq.rows;
      uint32_t qi, qg;
      a.shared.divmod(min(row0 + col, sq.rows - 1), qi, qg);
      const int64_t token = sq.q0 + qi;
      const int q_head = head * a.shared.d + qg;
      u32x4 q[NG];
      load_query<NG>(a, a.q + token * a.q_token + q_head * a.q_head, quad, q);
      const float top = in ? a.top[token * a.q_heads + q_head] : INFINITY;
      f32x4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
      for (int i = 0; i < NG; i++)
#pragma unroll
        for (int g = 0; g < 2; g++) acc[g] = mma<T>(k[g][i], q[i], acc[g]);
      const int sees = past + static_cast<int>(qi) - t - 4 * quad;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float w = __builtin_amdgcn_exp2f(
            __builtin_fmaf(acc[j >> 2][j & 3], a.scale_log2, -top));
        // (rows that see nothing have no weights, whatever their scores)
        sum[j] += sees >= 16 * (j >> 2) + (j & 3) && top != INFINITY ? w : 0.0f;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; j++)
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) sum[j] += __shfl_xor(sum[j], d);
    if (col < 8) {
      // lane `col` of a quarter has token 16 (col / 4) + 4 quad + col % 4
      float mine = sum[0];
#pragma unroll
      for (int j = 1; j < 8; j++) mine = col == j ? sum[j] : mine;
      const uint32_t own = static_cast<uint32_t>(t) + 16 * (col >> 2) + 4 * quad + (col & 3);
      if (own < static_cast<uint32_t>(sq.len)) {
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

// Workgroups that take the steps of a context in turn: one a step, fewer where there are very many.
uint32_t steps_of(int64_t max_len, int64_t contexts, int64_t heads) {
  const int64_t steps = (max_len + kStep - 1) / kStep;
  const int64_t most = (int64_t{1} << 20) / (contexts * heads) + 1;
  const int64_t n = steps < most ? steps : most;
  return static_cast<uint32_t>(n < 1 ? 1 : n);
}

}  // namespace

int full_weigh(const FullArgs& a, int type, int64_t max_len, int64_t max_prefix, hipStream_t s) {
  const FastDiv own(steps_of(max_len, a.own.n, a.heads));
  const FastDiv pre(a.pre.n > 0 ? steps_of(max_prefix, a.pre.n, a.heads) : 1);
  const int64_t prefix_items = static_cast<int64_t>(a.pre.n) * pre.d * a.heads;
  const int64_t items = prefix_items + static_cast<int64_t>(a.own.n) * own.d * a.heads;
  EVS_REQUIRE(items < (int64_t{1} << 23), "evs_attend: too many sequences and heads to weigh");
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
