// Attention over full-width pages for many query rows at a time (full.hpp has the mathematics).
#pragma once

#include "full_rows.hpp"

namespace evs {

// Tokens of a stage.
template <int NG>
constexpr int kStageTokens = NG > 4 ? 32 : 64;

template <int NG>
struct TilesLds {
  static constexpr int VD = Fetched<NG>::VD, VW = Fetched<NG>::VW;
  static constexpr int kSubs = kStageTokens<NG> / 32;
  // operands as the lanes read them, of this stage and the next
  // (K's chunks, of which a row has 4 NG, with a row's place among its 16 turned by the chunk's, so
  // that a row written and 16 rows read lie in different banks)
  u32x4 key[2][kSubs][2][NG][64];
  u32x4 value[2][kSubs][VD][VW][64];
  // ahead of the stages: their tokens' addresses, and which of them are tokens
  uint64_t at[4][kStageTokens<NG>];
  uint32_t ok[4][kSubs];
  uint32_t wild[4][kFullWaves];  // values that some rows see and some do not are no numbers
};

// A stage's rows on their way through registers to LDS: K as it lies, and V turned, so that a lane's
// operand is eight tokens' of one element. A wave has 16 tokens' K rows (of a stage of 32 tokens half
// of each), read row by row: read as operands, 16 bytes of 16 rows side by side, the chunks took the
// memory pipeline four times as long. A thread has, of eight tokens, half a chunk of V.
template <typename T, int NG, bool kWhole>
struct Staged {
  typedef TilesLds<NG> Lds;
  static constexpr int VD = Lds::VD, VW = Lds::VW, kSubs = Lds::kSubs;
  static constexpr int kKeys = NG * kSubs / 2;              // chunks of K that a thread has
  static constexpr int kWords = VW / 4;                     // dwords of a half chunk
  static_assert(kSubs * VD == 2, "");
  u32x4 k[kKeys];
  uint32_t v[8][2];

  // The row (of 16) and chunk that the lane's n-th load of K is of.
  static __device__ __forceinline__ void place(int n, int wave, int lane, int& row, int& chunk) {
    const int at = 64 * (kSubs == 2 ? n : kKeys * (wave / 2) + n) + lane;
    row = at / (4 * NG);
    chunk = at % (4 * NG);
  }

  // V: wave w has chunk column set (sub, v) = w / 2 and half w % 2.
  __device__ __forceinline__ void fetch(const FullArgs& a, const uint64_t* at, int wave, int lane) {
    const int col = lane & 15, quad = lane >> 4;
    const int rows16 = wave % (2 * kSubs);
#pragma unroll
    for (int n = 0; n < kKeys; n++) {
      int row, chunk;
      place(n, wave, lane, row, chunk);
      k[n] = load16(at[16 * rows16 + row] + 16 * (kWhole ? chunk : min(chunk, a.d / 8 - 1)));
    }
    const int sub = kSubs == 2 ? wave >> 1 : 0, vd = kSubs == 2 ? 0 : wave >> 1;
    const int e = min(VW * col + 128 * vd, a.d - VW) + VW / 2 * (wave & 1);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const uint64_t r = at[32 * sub + Fetched<NG>::token(j, quad)] + a.skv + 2 * e;
      if constexpr (kWords == 2) {
        const u32x2 x = load8(r);
        v[j][0] = x[0];
        v[j][1] = x[1];
      } else {
        v[j][0] = *reinterpret_cast<const __attribute__((address_space(1))) uint32_t*>(r);
      }
    }
  }

  // `tame`: some rows may not see all of the stage's tokens.
  __device__ __forceinline__ void store(const FullArgs& a, Lds& lds, int stage, int wave, int lane,
                                        bool tame) {
    const int quad = lane >> 4;
    const int rows16 = wave % (2 * kSubs);
#pragma unroll
    for (int n = 0; n < kKeys; n++) {
      int row, chunk;
      place(n, wave, lane, row, chunk);
      u32x4 x = k[n];
      // elements past the head size, which the query's zeros would meet, are to be numbers
      if (!kWhole && 8 * chunk >= a.d) x = u32x4{0, 0, 0, 0};
      lds.key[stage & 1][rows16 >> 1][rows16 & 1][chunk >> 2]
             [16 * (chunk & 3) + (row ^ (chunk & 15))] = x;
    }
    const int sub = kSubs == 2 ? wave >> 1 : 0, vd = kSubs == 2 ? 0 : wave >> 1;
    const uint32_t ok = __builtin_amdgcn_readfirstlane(lds.ok[stage & 3][sub]);
    bool wild = false;
    if (ok != 0xFFFFFFFFu || tame) {
      // rows of no tokens are to be numbers, whatever the pages hold: their weight is 0; so are
      // values that some rows see and some do not
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const bool in = (ok >> Fetched<NG>::token(j, quad)) & 1;
#pragma unroll
        for (int w = 0; w < kWords; w++) {
          v[j][w] = in ? v[j][w] : 0;
          if (tame) {
            wild |= is_wild<T>(v[j][w]);
            v[j][w] = tamed<T>(v[j][w]);
          }
        }
      }
    }
    const bool any = __builtin_amdgcn_ballot_w64(wild) != 0;
    if (lane == 0) lds.wild[stage & 3][wave] = any;
#pragma unroll
    for (int w = 0; w < kWords; w++) {
      u32x4 even, odd;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        even[j] = __builtin_amdgcn_perm(v[2 * j + 1][w], v[2 * j][w], 0x05040100u);
        odd[j] = __builtin_amdgcn_perm(v[2 * j + 1][w], v[2 * j][w], 0x07060302u);
      }
      const int e = VW / 2 * (wave & 1) + 2 * w;
      lds.value[stage & 1][sub][vd][e][lane] = even;
      lds.value[stage & 1][sub][vd][e + 1][lane] = odd;
    }
  }
};

// One workgroup: part `item` of the contexts of tiles of 64 * kTiles query rows and one KV head,
// 16 * kTiles rows a wave, which all take every token of a stage.
//
// Bound by the matrix instructions and, beside them, each score's exponential and packing: a stage of
// tokens is read once for all rows of the tile, into registers while the stage before is computed.
// Four chunks of 1,024 queries at the end of 4 to 8 Ki tokens, 32 heads of 128 on 8: 425 us, 848
// TFLOP/s (a large library product: 1,197); one prompt of 4,096 from its start 192 us, 718 TFLOP/s. Of
// few sequences a workgroup's stages are a chain of 1.7 us each, 2.3 with two workgroups a CU.
template <typename T, int NG, bool kWhole, int kTiles>
__device__ __forceinline__ void tiles_part(const FullArgs& a, TilesLds<NG>& lds, uint32_t item,
                                           uint32_t prefix_items) {
  typedef TilesLds<NG> Lds;
  constexpr int VD = Lds::VD, VW = Lds::VW, kSubs = Lds::kSubs;
  constexpr int kTokens = kStageTokens<NG>;
  constexpr int kRows = 16 * kTiles * kFullWaves;

  // which rows, which part of which context
  const bool prefix = item < prefix_items;
  const Cut& cut = prefix ? a.group : a.many;
  uint32_t at = prefix ? item : item - prefix_items;
  // Workgroups go to the 8 XCDs in turn: all row tiles of a head and part to one, whose rows then
  // stay in its L2.
  const uint32_t unit = at / (8 * cut.tiles) * 8 + (at & 7);
  // (the last first: of a sequence's tiles they see the most tokens)
  const uint32_t place = cut.tiles - 1 - (at >> 3) % cut.tiles;
  uint32_t head, split, who, tile;
  a.div_heads.divmod(unit, split, head);
  if (static_cast<int>(split) >= cut.splits) return;
  Rows sq;
  const auto tiles_of = [&](const Rows& r) -> uint32_t {
    return prefix || r.rows > kRowTile ? (r.rows + kRows - 1) / kRows : 0;
  };
  if (prefix ? !find_rows(a.pre.n, place, [&](uint32_t i) { return group_rows(a, i); }, tiles_of,
                          who, tile, sq)
             : !find_rows(a.own.n, place, [&](uint32_t i) { return sequence_rows(a, i); }, tiles_of,
                          who, tile, sq))
    return;
  const int row0 = tile * kRows, last_row = min(row0 + kRows, sq.rows) - 1;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, quad = lane >> 4;
  bool needed = true;  // this wave's rows
  int ahead_len = 0;   // tokens of a prefix ahead of the own ones
  const int32_t* ahead_table = nullptr;
  if (prefix) {
    if (a.starts != nullptr && a.max_q * static_cast<int>(a.shared.d) > kTogether) {
      // only for rows of sequences that take their prefix with the group
      const int from = sq.q0 + static_cast<int>(a.shared.div(row0));
      const int to = sq.q0 + static_cast<int>(a.shared.div(last_row));
      const int s0 = min(max(a.group_starts[who], 0), a.seqs);
      const int s1 = min(max(a.group_starts[who + 1], s0), a.seqs);
      const int wave_from = sq.q0 + static_cast<int>(a.shared.div(row0 + 16 * kTiles * wave));
      const int wave_to = sq.q0 + static_cast<int>(a.shared.div(row0 + 16 * kTiles * (wave + 1) - 1));
      bool any = false, mine = false;
      for (int s = s0 + lane; s < s1; s += 64) {
        const Rows r = sequence_rows(a, s);
        const bool with = r.rows > 0 && r.rows <= kTogether;
        any |= with && r.q0 <= to && r.q0 + r.nq > from;
        mine |= with && r.q0 <= wave_to && r.q0 + r.nq > wave_from;
      }
      if (__builtin_amdgcn_ballot_w64(any) == 0) return;
      needed = __builtin_amdgcn_ballot_w64(mine) != 0;
    }
  } else if (sq.rows > kTogether) {
    const int g = group_of(a, who);
    if (g >= 0) {
      ahead_len = __builtin_amdgcn_readfirstlane(length_of(a, a.pre, g));
      ahead_table = a.pre.tables + static_cast<int64_t>(g) * a.pre.stride;
    }
  }
  const int len = ahead_len + sq.len;
  // own tokens are seen up to the query's own, a prefix by every row
  const int past = prefix ? len : len - sq.nq;
  const auto seen_by = [&](int row) {  // the tokens that a row sees
    return min(len, max(past + static_cast<int>(a.shared.div(row)) + 1, ahead_len));
  };
  const int end = seen_by(last_row);
  const int begin = split * cut.chunk;
  const int stop =
      static_cast<int>(split) + 1 == cut.splits ? end : min(end, begin + cut.chunk);
  if (begin >= stop && (prefix || split > 0)) return;
  const int stages = stop > begin ? (stop - begin + kTokens - 1) / kTokens : 0;

  // this wave's rows, and the tokens that some and all of them see
  const int wave0 = row0 + 16 * kTiles * wave;
  const bool any_row = needed && wave0 <= last_row;
  const int wave_stop =
      any_row ? min(stop, seen_by(min(wave0 + 16 * kTiles - 1, last_row))) : 0;
  const int all_see = any_row ? min(stop, seen_by(wave0)) : 0;
  const int tile_see = min(stop, seen_by(row0));
  int sees[kTiles];
  const char* qp[kTiles];
#pragma unroll
  for (int n = 0; n < kTiles; n++) {
    uint32_t qi, qg;
    a.shared.divmod(min(wave0 + 16 * n + col, last_row), qi, qg);
    sees[n] = max(past + static_cast<int>(qi), ahead_len - 1);
    qp[n] = a.q + (sq.q0 + qi) * a.q_token + (head * a.shared.d + qg) * a.q_head;
  }
  const int32_t* table = prefix ? a.pre.tables + static_cast<int64_t>(who) * a.pre.stride
                                : a.own.tables + static_cast<int64_t>(who) * a.own.stride;
  const uint64_t base = reinterpret_cast<uint64_t>(a.base) + head * a.sh;

  f32x4 o[kTiles][VD][VW];
#pragma unroll
  for (int n = 0; n < kTiles; n++)
#pragma unroll
    for (int v = 0; v < VD; v++)
#pragma unroll
      for (int j = 0; j < VW; j++) o[n][v][j] = f32x4{0, 0, 0, 0};
  Running run[kTiles];

  if (stages > 0) {
    // (without a sign: past the last stage it may pass 2^31)
    const auto token_of = [&](int stage) {
      return min(static_cast<uint32_t>(begin) + static_cast<uint32_t>(stage * kTokens + tid),
                 static_cast<uint32_t>(stop) - 1);
    };
    // the page of the thread's token of a stage, read a stage before its address is needed
    const auto page_of = [&](int stage) {
      const uint32_t t = token_of(stage);
      const bool early = t < static_cast<uint32_t>(ahead_len);
      return (early ? ahead_table : table)[a.div_bs.div(early ? t : t - ahead_len)];
    };
    // the tokens' addresses and flags, by as many threads
    const auto locate = [&](int stage, int32_t page) {
      if (tid < kTokens) {
        const uint32_t t = token_of(stage);
        const bool ok = static_cast<uint32_t>(begin) + static_cast<uint32_t>(stage * kTokens + tid) <
                            static_cast<uint32_t>(stop) &&
                        page >= 0 && page < a.num_blocks;
        uint32_t n, off;
        a.div_bs.divmod(t < static_cast<uint32_t>(ahead_len) ? t : t - ahead_len, n, off);
        lds.at[stage & 3][tid] = base + (ok ? page * a.sb + static_cast<int64_t>(off) * a.so : 0);
        const unsigned long long flags = __builtin_amdgcn_ballot_w64(ok);
        if ((tid & 31) == 0)
          lds.ok[stage & 3][tid >> 5] = static_cast<uint32_t>(flags >> (tid & 32));
      }
    };
    int32_t pages[3];
#pragma unroll
    for (int k = 0; k < 3; k++) pages[k] = page_of(k);
    int32_t page = page_of(3);
    u32x4 q[kTiles][NG];
#pragma unroll
    for (int n = 0; n < kTiles; n++) load_query<NG>(a, qp[n], quad, q[n]);
#pragma unroll
    for (int k = 0; k < 3; k++) locate(k, pages[k]);
    __syncthreads();
    const auto tame = [&](int stage) {  // (its end may pass 2^31)
      return static_cast<uint32_t>(begin) + static_cast<uint32_t>((stage + 1) * kTokens) >
             static_cast<uint32_t>(tile_see);
    };
    Staged<T, NG, kWhole> rows;
    rows.fetch(a, lds.at[0], wave, lane);
    rows.store(a, lds, 0, wave, lane, tame(0));
    rows.fetch(a, lds.at[1], wave, lane);

    // Stage i is computed with while the rows of the next are written to LDS and those of the one
    // after are on their way: one barrier a stage. (Past the last stage the last token's page is
    // read.)
    for (int i = 0; i < stages; i++) {
      __syncthreads();
      rows.store(a, lds, i + 1, wave, lane, tame(i + 1));
      locate(i + 3, page);
      page = page_of(i + 4);
      rows.fetch(a, lds.at[(i + 2) & 3], wave, lane);
      const int t0 = begin + i * kTokens;
      if (t0 >= wave_stop) continue;
      const bool wild = __builtin_amdgcn_ballot_w64(lds.wild[i & 3][lane & (kFullWaves - 1)] != 0) != 0;
      f32x4 acc[kSubs][2][kTiles];
#pragma unroll
      for (int sub = 0; sub < kSubs; sub++)
#pragma unroll
        for (int g = 0; g < 2; g++)
#pragma unroll
          for (int n = 0; n < kTiles; n++) acc[sub][g][n] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int sub = 0; sub < kSubs; sub++)
#pragma unroll
        for (int c = 0; c < NG; c++)
#pragma unroll
          for (int g = 0; g < 2; g++) {
            const u32x4 k = lds.key[i & 1][sub][g][c][lane ^ ((4 * c + quad) & 15)];
#pragma unroll
            for (int n = 0; n < kTiles; n++) acc[sub][g][n] = mma<T>(k, q[n][c], acc[sub][g][n]);
          }
      float s[kTiles][8 * kSubs];
#pragma unroll
      for (int n = 0; n < kTiles; n++)
#pragma unroll
        for (int k = 0; k < 8 * kSubs; k++) s[n][k] = acc[k >> 3][(k >> 2) & 1][n][k & 3];
      uint32_t ok[kSubs], all = 0xFFFFFFFFu;
#pragma unroll
      for (int sub = 0; sub < kSubs; sub++) {
        ok[sub] = __builtin_amdgcn_readfirstlane(lds.ok[i & 3][sub]);
        all &= ok[sub];
      }
      if (__builtin_expect(t0 > all_see - kTokens || all != 0xFFFFFFFFu, false)) {
        asm volatile("");  // a branch: most stages need none of it
#pragma unroll
        for (int sub = 0; sub < kSubs; sub++)
#pragma unroll
          for (int k = 0; k < 8; k++) {
            const int at = 16 * (k >> 2) + 4 * quad + (k & 3);
            const bool in = (ok[sub] >> at) & 1;
#pragma unroll
            for (int n = 0; n < kTiles; n++)
              s[n][8 * sub + k] =
                  in && t0 + 32 * sub + at <= sees[n] ? s[n][8 * sub + k] : -INFINITY;
          }
      }
      float fade[kTiles];
      if (grow<kTiles>(s, a.scale_log2, run, fade)) {
#pragma unroll
        for (int n = 0; n < kTiles; n++)
#pragma unroll
          for (int v = 0; v < VD; v++)
#pragma unroll
            for (int j = 0; j < VW; j++) o[n][v][j] *= fade[n];
      }
      if (__builtin_expect(wild, false)) {
#pragma unroll
        for (int sub = 0; sub < kSubs; sub++)
#pragma unroll
          for (int n = 0; n < kTiles; n++)
            add_wild<T, VW, VD>(a, lds.at[i & 3] + 32 * sub, ok[sub], sees[n] - t0 - 32 * sub,
                                &s[n][8 * sub], run[n], o[n]);
      }
      u32x4 p[kSubs][kTiles];
#pragma unroll
      for (int sub = 0; sub < kSubs; sub++)
#pragma unroll
        for (int n = 0; n < kTiles; n++)
          p[sub][n] = full_weights<T>(&s[n][8 * sub], a.scale_log2, run[n]);
#pragma unroll
      for (int sub = 0; sub < kSubs; sub++)
#pragma unroll
        for (int v = 0; v < VD; v++)
#pragma unroll
          for (int j = 0; j < VW; j++) {
            const u32x4 x = lds.value[i & 1][sub][v][j][lane];
#pragma unroll
            for (int n = 0; n < kTiles; n++) o[n][v][j] = mma<T>(x, p[sub][n], o[n][v][j]);
          }
    }
  }

  // Element VW (4 quad + r) + j, from 128 v on, of row `col` of a tile is o[n][v][j][r].
  const int slot = prefix ? split : a.group.splits + split;
  const bool joined = prefix || is_joined(a, cut, sq.rows, end);
#pragma unroll
  for (int n = 0; n < kTiles; n++) {
    const float l = across_rows_sum(run[n].l);
    const int row = wave0 + 16 * n + col;
    if (!any_row || row > last_row) continue;
    uint32_t i, g;
    a.shared.divmod(row, i, g);
#pragma unroll
    for (int v = 0; v < VD; v++)
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int j = 0; j < VW; j += 4) {
          const int e = 128 * v + VW * (4 * quad + r) + j;
          if (e >= a.d) continue;
          const f32x4 x = {o[n][v][j][r], o[n][v][j + 1][r], o[n][v][j + 2][r], o[n][v][j + 3][r]};
          const int token = sq.q0 + i, q_head = head * a.shared.d + g;
          if (joined)
            keep4(a.parts, a.d, part_at(a, slot, token, q_head), e / 4, x, run[n].m, l);
          else
            finish4<T>(a, token, q_head, e / 4, x, run[n].m, l);
        }
  }
}

}  // namespace evs
