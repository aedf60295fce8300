// Attention over full-width pages for few query rows at a time (full.hpp has the mathematics).
#pragma once

#include "full.hpp"

namespace evs {

// 32 tokens' rows, as a wave's lanes have them: K as operands as they lie, and of V eight tokens'
// chunk of VW elements, which are turned within the lane. kWhole: the head size is 32 NG, so that
// every chunk's offset is a constant.
template <int NG>
struct Fetched {
  static constexpr int VD = NG > 4 ? 2 : 1;  // chunks of a V row that a lane has
  static constexpr int VW = NG > 2 ? 8 : 4;  // elements of a chunk
  typedef typename std::conditional<VW == 8, u32x4, u32x2>::type Chunk;
  u32x4 k[2][NG];
  Chunk v[8][VD];

  // Token of the 32 whose V chunk is v[j].
  static __device__ __forceinline__ int token(int j, int quad) {
    return 16 * (j >> 2) + 4 * quad + (j & 3);
  }

  template <bool kWhole>
  __device__ __forceinline__ void fetch_keys(const FullArgs& a, const uint64_t* at, int lane) {
    const int col = lane & 15, quad = lane >> 4;
#pragma unroll
    for (int g = 0; g < 2; g++) {
      const uint64_t p = at[16 * g + col];
#pragma unroll
      for (int i = 0; i < NG; i++)
        k[g][i] = load16(kWhole ? p + 16 * quad + 64 * i : p + 16 * min(4 * i + quad, a.d / 8 - 1));
    }
  }

  __device__ __forceinline__ void fetch_values(const FullArgs& a, const uint64_t* at, int lane) {
    const int col = lane & 15, quad = lane >> 4;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const uint64_t p = at[token(j, quad)] + a.skv;
#pragma unroll
      for (int v = 0; v < VD; v++) {
        const int e = min(VW * col + 128 * v, a.d - VW);
        if constexpr (VW == 8)
          this->v[j][v] = load16(p + 2 * e);
        else
          this->v[j][v] = load8(p + 2 * e);
      }
    }
  }

  // The elements of K past the head size, which the query's zeros would meet, are to be numbers.
  __device__ __forceinline__ void trim(const FullArgs& a, int quad) {
#pragma unroll
    for (int i = 0; i < NG; i++)
      if (32 * (i + 1) > a.d) {
        const bool in = 8 * (4 * i + quad) < a.d;
#pragma unroll
        for (int g = 0; g < 2; g++)
#pragma unroll
          for (int k = 0; k < 4; k++) this->k[g][i][k] = in ? this->k[g][i][k] : 0;
      }
  }
};

template <int NG>
union RowsLds {
  uint64_t at[kFullWaves][2][64];  // a wave's tokens' addresses, 64 at a time
  struct {
    float o[kFullWaves][kRowTile][16 * Fetched<NG>::VW * Fetched<NG>::VD + 4];
    float m[kFullWaves][kRowTile], l[kFullWaves][kRowTile];
  } joined;
};

// One workgroup: part `item` of the contexts of tiles of 16 query rows and one KV head, 64 tokens of
// it a wave in turn. Nothing passes through LDS but the tokens' addresses and the waves' results.
// Each wave has kSets times 32 tokens' rows under way.
//
// Bound by the cache's bytes, which pass from memory to registers and are used there once: K is an
// operand as it lies, V is turned within the lane. 64 sequences of 1 to 4 Ki tokens, 8 KV heads of 128,
// four query heads each: 143 us, 4.7 TB/s (16 Ki tokens: 5.1 TB/s), two workgroups a CU; more rows
// under way gained nothing, and the registers of a third workgroup spill. A short context's time is the
// launch and a chain of reads, lengths, pages, rows: 600 tokens 12 us.
template <typename T, int NG, bool kWhole, int kSets>
__device__ __forceinline__ void rows_part(const FullArgs& a, RowsLds<NG>& lds, uint32_t item,
                                          uint32_t prefix_items) {
  typedef Fetched<NG> Rows32;
  constexpr int VD = Rows32::VD, VW = Rows32::VW;

  // which rows, which part of which context
  const bool prefix = item < prefix_items;
  const Contexts& c = prefix ? a.pre : a.own;
  const Cut& cut = prefix ? a.group : a.few;
  uint32_t head, rest, who, split;
  a.div_heads.divmod(prefix ? item : item - prefix_items, rest, head);
  split = rest / cut.tiles;
  who = rest - split * cut.tiles;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t* table = c.tables + static_cast<int64_t>(who) * c.stride;
  const int begin = split * cut.chunk;
  const int first = begin + 64 * wave;
  constexpr int step = 64 * kFullWaves;
  // The first pages are read ahead of the length, which they do not wait for; so tokens are kept
  // within the table, and what lies past the length is no token. (Without a sign: past the last
  // pair a token may pass 2^31.)
  const uint32_t room = static_cast<uint32_t>(
      min(static_cast<int64_t>(c.width) * a.block_size, (int64_t{1} << 31) - 1));
  const auto token_of = [&](int p) {
    return static_cast<uint32_t>(first) + static_cast<uint32_t>(p * step + lane);
  };
  const auto page_of = [&](int p) {
    return room == 0 ? -1 : table[a.div_bs.div(min(token_of(p), room - 1))];
  };
  int32_t page = page_of(0), page_next = page_of(1);
  const Rows sq = scalar_rows(prefix ? group_rows(a, who) : sequence_rows(a, who));
  if (sq.rows == 0 || sq.rows > kRowTile) return;
  const int last_row = sq.rows - 1;
  // own tokens are seen up to the query's own, a prefix by every row
  const int past = prefix ? sq.len : sq.len - sq.nq;
  const int end = prefix ? sq.len : min(sq.len, past + sq.nq);
  const int stop =
      static_cast<int>(split) + 1 == cut.splits ? end : min(end, begin + cut.chunk);
  if (begin >= stop && (prefix || split > 0)) return;

  const int col = lane & 15, quad = lane >> 4;
  uint32_t qi, qg;
  a.shared.divmod(min(col, last_row), qi, qg);
  const int sees = past + static_cast<int>(qi);  // this lane's row: the tokens up to this one
  const int all_see = min(stop, past + 1);
  const uint64_t base = reinterpret_cast<uint64_t>(a.base) + head * a.sh;

  f32x4 o[VD][VW];
#pragma unroll
  for (int v = 0; v < VD; v++)
#pragma unroll
    for (int j = 0; j < VW; j++) o[v][j] = f32x4{0, 0, 0, 0};
  Running run[1];

  // (token t's score with this lane's row goes to scores[t])
  float* scores = prefix || a.scores == nullptr
                      ? nullptr
                      : a.scores + few_part_at(a, 0, who, head, min(col, last_row)) * a.stored;

  if (first < stop) {
    const int pairs = (stop - first + step - 1) / step;
    // the addresses of a pair's tokens, and which of them are tokens
    const auto locate = [&](int p, int32_t page) {
      const uint32_t t = token_of(p);
      uint32_t n, off;
      a.div_bs.divmod(min(t, room - 1), n, off);
      const bool ok = t < static_cast<uint32_t>(stop) && page >= 0 && page < a.num_blocks;
      wave_sync();  // those before have been read
      lds.at[wave][p & 1][lane] = base + (ok ? page * a.sb + static_cast<int64_t>(off) * a.so : 0);
      wave_sync();  // other lanes of the wave read them
      return __builtin_amdgcn_ballot_w64(ok);
    };
    u32x4 q[NG];
    load_query<NG>(a, a.q + (sq.q0 + qi) * a.q_token + (head * a.shared.d + qg) * a.q_head, quad,
                   q);
    unsigned long long ok = locate(0, page), ok_next = 0;
    page = page_next;
    Rows32 rows[kSets];
#pragma unroll
    for (int n = 0; n < kSets; n++) {
      rows[n].template fetch_keys<kWhole>(a, lds.at[wave][0] + 32 * n, lane);
      rows[n].fetch_values(a, lds.at[wave][0] + 32 * n, lane);
    }
    for (int p = 0; p < pairs; p++) {
      ok_next = locate(p + 1, page);
      page = page_of(p + 2);
#pragma unroll
      for (int sub = 0; sub < 2; sub++) {
        Rows32& x = rows[sub % kSets];
        // what is fetched next into the same registers
        const uint64_t* next =
            sub + kSets < 2 ? &lds.at[wave][p & 1][32] : &lds.at[wave][(p + 1) & 1][kSets == 1 ? 0 : 32 * sub];
        const int t = first + p * step + 32 * sub;
        const uint32_t there = static_cast<uint32_t>(ok >> (32 * sub));
        if (!kWhole) x.trim(a, quad);
        f32x4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int i = 0; i < NG; i++)
#pragma unroll
          for (int g = 0; g < 2; g++) acc[g] = mma<T>(x.k[g][i], q[i], acc[g]);
        x.template fetch_keys<kWhole>(a, next, lane);
        float s[1][8];
#pragma unroll
        for (int k = 0; k < 8; k++) s[0][k] = acc[k >> 2][k & 3];
        // (t + 32 may pass 2^31)
        const bool whole = t <= all_see - 32 && there == 0xFFFFFFFFu;
        bool wild = false;
        if (__builtin_expect(!whole, false)) {
          asm volatile("");  // a branch: most tokens need none of it
          const int ahead[1] = {sees - t - 4 * quad};
          mask<1>(s, ahead, there >> (4 * quad));
          // rows of no tokens are to be numbers, whatever the pages hold: their weight is 0; so
          // are values that some rows see and some do not
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const bool in = (there >> Rows32::token(j, quad)) & 1;
#pragma unroll
            for (int v = 0; v < VD; v++)
#pragma unroll
              for (int k = 0; k < VW / 2; k++) {
                x.v[j][v][k] = in ? x.v[j][v][k] : 0;
                wild |= is_wild<T>(x.v[j][v][k]);
              }
          }
          wild = t > all_see - 32 && __builtin_amdgcn_ballot_w64(wild) != 0;
        }
        float fade[1];
        if (grow<1>(s, a.scale_log2, run, fade)) {
#pragma unroll
          for (int v = 0; v < VD; v++)
#pragma unroll
            for (int j = 0; j < VW; j++) o[v][j] *= fade[0];
        }
        if (__builtin_expect(wild, false)) {
#pragma unroll
          for (int j = 0; j < 8; j++)
#pragma unroll
            for (int v = 0; v < VD; v++)
#pragma unroll
              for (int k = 0; k < VW / 2; k++) x.v[j][v][k] = tamed<T>(x.v[j][v][k]);
          add_wild<T, VW, VD>(a, lds.at[wave][p & 1] + 32 * sub, there, sees - t, s[0], run[0], o);
        }
        const u32x4 w = full_weights<T>(s[0], a.scale_log2, run[0]);
        // eight tokens' elements 2c and 2c + 1, side by side
#pragma unroll
        for (int v = 0; v < VD; v++)
#pragma unroll
          for (int k = 0; k < VW / 2; k++) {
            u32x4 even, odd;
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const uint32_t lo = x.v[2 * j][v][k], hi = x.v[2 * j + 1][v][k];
              even[j] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
              odd[j] = __builtin_amdgcn_perm(hi, lo, 0x07060302u);
            }
            o[v][2 * k] = mma<T>(even, w, o[v][2 * k]);
            o[v][2 * k + 1] = mma<T>(odd, w, o[v][2 * k + 1]);
          }
        x.fetch_values(a, next, lane);
        // behind the loads: waiting for those is not to wait for this
        if (scores != nullptr && col < sq.rows) {
#pragma unroll
          for (int g = 0; g < 2; g++) {
            const uint32_t at = static_cast<uint32_t>(t) + 16 * g + 4 * quad;
            if (at < static_cast<uint32_t>(a.stored))
              *reinterpret_cast<f32x4*>(scores + at) = acc[g];
          }
        }
      }
      ok = ok_next;
    }
  }
  run[0].l = across_rows_sum(run[0].l);

  // Element VW (4 quad + r) + j, from 128 v on, of row `col` is o[v][j][r].
  __syncthreads();  // the addresses have been read
#pragma unroll
  for (int v = 0; v < VD; v++)
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
      for (int j = 0; j < VW; j += 4)
        *reinterpret_cast<f32x4*>(
            &lds.joined.o[wave][col][128 * v + VW * (4 * quad + r) + j]) =
            f32x4{o[v][j][r], o[v][j + 1][r], o[v][j + 2][r], o[v][j + 3][r]};
  if (quad == 0) {
    lds.joined.m[wave][col] = run[0].m;
    lds.joined.l[wave][col] = run[0].l;
  }
  __syncthreads();
  const int words = a.d / 4;
  const bool joined = prefix || is_joined(a, a.few, sq.rows, end);
  for (int x = threadIdx.x; x < sq.rows * words; x += kFullThreads) {
    const int r = x / words, w = x - r * words;
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < kFullWaves; k++) top = fmaxf(top, lds.joined.m[k][r]);
    const float ref = top == -INFINITY ? 0.0f : top;
    float total = 0;
    f32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < kFullWaves; k++) {
      const float f = __builtin_amdgcn_exp2f(lds.joined.m[k][r] - ref);
      total += f * lds.joined.l[k][r];
      v += f * *reinterpret_cast<const f32x4*>(&lds.joined.o[k][r][4 * w]);
    }
    uint32_t i, g;
    a.shared.divmod(r, i, g);
    const int token = sq.q0 + i, q_head = head * a.shared.d + g;
    if (prefix)
      keep4(a.parts, a.d, part_at(a, split, token, q_head), w, v, top, total);
    else if (joined)
      keep4(a.few_parts, a.d, few_part_at(a, split, who, head, r), w, v, top, total);
    else
      finish4<T>(a, token, q_head, w, v, top, total);
    if (!joined && a.scores != nullptr && w == 0) {
      // the weights' references
      float* stats = a.few_parts.stats + 2 * few_part_at(a, split, who, head, r);
      stats[0] = top;
      stats[1] = total;
    }
  }
}

}  // namespace evs
