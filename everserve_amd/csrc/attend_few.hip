// Attention over 4-bit pages for sequences with few query rows: single tokens, and a few at once
// (attend.hpp has the mathematics).
#include "attend.hpp"

namespace evs {
namespace {

constexpr int kTile = 32;  // tokens a wave takes at once

// One workgroup: a share of the stages of tiles of 16 query rows, for a group of KV heads whose
// rows lie side by side. A stage is 32 tokens of every wave's head; waves with one head take a
// stage's tokens in turns of 32 and join their results in LDS.
//
// Bound by reading pages at random places. 64 sequences of 1 to 8 Ki tokens, 32 heads on 8 of 128,
// 322 MB: 76 us, 4.2 TB/s (a loop that only fetches the same rows took 63, 5.1; a large plain copy
// reaches 4.84 and a plain read 6.3). About 8 us of it are the start, in which three loads wait for
// each other (a length, page ids, rows). So:
// - a stage's rows are fetched by all waves together, a token's heads in one run of memory, into
//   registers, two stages before their use, and pass through LDS with one barrier a stage (fetched
//   by each wave for its own head: 84 us);
// - one workgroup a CU with the registers of two, for heads above 64: two leave room for one stage
//   under way (the call of the decode step above 80 us for 78, with f16 queries 112 for 87; where
//   a page has a head's rows together, `combined`, 85 for 91 and 118 for 106);
// - codes become bf16 operands in registers, right before the products; a tile is 16 rows, as wide
//   as an MFMA, since there are mostly fewer.
template <int NG, bool kWhole, typename T>
__global__ __launch_bounds__(64 * kFewWaves, NG > 2 ? 2 : 4) void attend_rows(AttendArgs a) {
  constexpr int kTerms = QueryTerms<T>::n;
  constexpr int VD = NG > 4 ? 2 : 1;  // dwords of V a lane holds of a token
  // stages whose rows are on their way; wide rows leave no registers for a second
  constexpr int kAhead = NG > 4 ? 1 : 2;
  typedef Stage<NG, kTile, kFewWaves, kWhole> Rows;
  struct Joined {
    float o[kFewWaves][kFewTile][128 * VD + 4];
    float m[kFewWaves][kFewTile], l[kFewWaves][kFewTile];
  };
  union Shared {
    typename Rows::Lds rows[2];  // of this stage and the next
    Joined joined;
  };
  __shared__ Shared lds;
  __shared__ typename Rows::Tokens tk;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Workgroups go to the 8 XCDs in turn: a share's groups, whose rows share memory lines, to one.
  uint32_t group, outer;
  a.groups.divmod(blockIdx.x >> 3, outer, group);
  const uint32_t owner = 8 * outer + (blockIdx.x & 7);
  const uint32_t held = a.held.d;
  uint32_t h, turn;
  a.held.divmod(wave, turn, h);
  const uint32_t head = group * held + h;
  const int tokens = kTile * a.turns;  // of a stage
  const char* base = a.c.base + static_cast<int64_t>(group * held) * a.c.sh;
  Share share;
  if (!find_share<false>(args_now(), owner, tokens, share)) return;
  Sequence sq = sequence_of_all(a, share.seq);

  while (true) {
    const int lane = lane_now();
    const int col = lane & 15, quad = lane >> 4;
    const Part part = next_part<false>(args_now(), sq, share, tokens);
    if (part.none) return;
    if (part.slot == 1 && group == 0 && threadIdx.x == 0) {
      const AttendArgs b = args_now();
      if (b.few.split) describe<false>(b, share, owner, part);
    }
    // this lane's query row, and the tokens that it sees: those up to `sees`
    uint32_t qi, qg;
    a.shared.divmod(min(part.row0 + col, part.last_row), qi, qg);
    const int past = sq.len - sq.nq;
    const int sees = past + static_cast<int>(qi);
    // tokens that all of the rows see
    const int begin = part.begin, stop = part.stop;
    const int all_see = min(stop, past + static_cast<int>(a.shared.div(part.row0)) + 1);
    const int stages = stop > begin ? (stop - begin + tokens - 1) / tokens : 0;
    const int32_t* table = a.tables + static_cast<int64_t>(share.seq) * a.table_stride;

    f32x4 o[VD][8];
#pragma unroll
    for (int v = 0; v < VD; v++)
#pragma unroll
      for (int j = 0; j < 8; j++) o[v][j] = f32x4{0, 0, 0, 0};
    Running run[1];

    if (stages > 0) {
      Rows rows;
      rows.place(a, wave, lane, a.held, tokens);
      const int tid = 64 * wave + lane;
      // (without a sign: past the last stage it may pass 2^31)
      const auto token_of = [&](int stage) {
        return static_cast<uint32_t>(begin) + static_cast<uint32_t>(stage * tokens + tid);
      };
      const auto page_of = [&](int stage) {
        return Rows::page_of(a, table, token_of(stage), stop);
      };
      const auto locate = [&](int stage, int32_t page) {
        if (64 * wave < tokens)
          Rows::locate(a, tk, stage, base, token_of(stage), stop, page, tid, tokens);
      };
      int32_t pages[4];
#pragma unroll
      for (int k = 0; k < 4; k++) pages[k] = page_of(k);
      int32_t page = page_of(4);
#pragma unroll
      for (int k = 0; k < 4; k++) locate(k, pages[k]);
      __syncthreads();
      Rows other = rows;
      other.fetch(a, tk.at[0], lane);
      if (kAhead == 2) rows.fetch(a, tk.at[1], lane);
      Query<NG, T> q[1];
      q[0].load(a, a.q + (sq.q0 + qi) * a.q_token + (head * a.shared.d + qg) * a.q_head, quad);

      const uint32_t row = h * tokens + kTile * turn;  // this wave's first row of a stage
      int vw[VD];
#pragma unroll
      for (int v = 0; v < VD; v++) vw[v] = min(16 * v + col, a.c.W - 1);

      other.store(a, lds.rows[0], tk, 0, wave, lane);
      if (kAhead == 2)
        other.fetch(a, tk.at[2], lane);
      else
        rows.fetch(a, tk.at[1], lane);

      // Stage i is computed with while the rows of the next are written to LDS, those after are on
      // their way and those of one more are located: one barrier a stage. (Past the last stage the
      // last token's page is read.)
      const auto take = [&](int i, Rows& next) {
        __syncthreads();
        next.store(a, lds.rows[(i + 1) & 1], tk, i + 1, wave, lane);
        locate(i + 4, page);
        page = page_of(i + 5);
        next.fetch(a, tk.at[(i + 1 + kAhead) & 3], lane);
        const typename Rows::Lds& now = lds.rows[i & 1];

        const int t = begin + i * tokens + kTile * static_cast<int>(turn);
        if (t < stop) {
          f32x4 acc[2][1];
          scores<NG, 1, T>(now, row, lane, a.c.W, q, acc);
          float s[1][8];
#pragma unroll
          for (int k = 0; k < 8; k++) s[0][k] = acc[k >> 2][0][k & 3];
          const uint32_t ok = __builtin_amdgcn_readfirstlane(tk.ok[i & 7][turn]);
          const bool whole = t + kTile <= all_see && ok == 0xFFFFFFFFu;
          bool wild = false;
          if (!whole) {
            const int ahead[1] = {sees - t - 4 * quad};
            mask<1>(s, ahead, ok >> (4 * quad));
            wild = __builtin_amdgcn_ballot_w64(
                       tk.wild[i & 3][min(lane, static_cast<int>(held * a.turns) - 1)] != 0) != 0;
          }
          float fade[1];
          if (grow<1>(s, a.scale_log2, run, fade)) {
#pragma unroll
            for (int v = 0; v < VD; v++)
#pragma unroll
              for (int j = 0; j < 8; j++) o[v][j] *= fade[0];
          }
          if (wild) {
#pragma unroll
            for (int v = 0; v < VD; v++)
              add_wild(now, row, v, a.c.W, sees - t, ok, s[0], a.scale_log2, run[0], o[v]);
          }
          u32x4 p[kTerms];
          weights<kTerms>(s[0], a.scale_log2, run[0], p);
#pragma unroll
          for (int v = 0; v < VD; v++) {
            Values x;
            x.load(now, row, quad, vw[v]);
            float sc[8];
            x.to_f32(sc);
            if (wild) tame(x.codes, sc);
            const auto pair = [&](auto c_) {
              constexpr int c = decltype(c_)::value;
              bf16x8 even, odd;
              value_pair<c>(x.codes, sc, even, odd);
#pragma unroll
              for (int n = 0; n < kTerms; n++) {
                const bf16x8 pf = __builtin_bit_cast(bf16x8, p[n]);
                o[v][2 * c] =
                    __builtin_amdgcn_mfma_f32_16x16x32_bf16(even, pf, o[v][2 * c], 0, 0, 0);
                o[v][2 * c + 1] =
                    __builtin_amdgcn_mfma_f32_16x16x32_bf16(odd, pf, o[v][2 * c + 1], 0, 0, 0);
              }
            };
            pair(std::integral_constant<int, 0>{});
            pair(std::integral_constant<int, 1>{});
            pair(std::integral_constant<int, 2>{});
            pair(std::integral_constant<int, 3>{});
          }
        }
      };
      for (int i = 0; i < stages; i += kAhead) {
        take(i, rows);
        if (kAhead == 2 && i + 1 < stages) take(i + 1, other);
      }
      __syncthreads();  // the rows have been read
    }
    run[0].l = across_rows_sum(run[0].l);

    {
    const AttendArgs b = args_now();
    const uint32_t held = b.held.d;
    const int lane = lane_now();
    const int col = lane & 15, quad = lane >> 4;
    // Element 8 (4 quad + r) + j of row `col` is o[v][j][r].
    const auto put = [&](uint32_t at, int r, int w, const float (&x)[8], float top, float total) {
      if (part.whole)
        finish<T>(b, sq, part.row0 + r, at, w, x, top, total);
      else
        keep(b, part_row(b, b.few, owner, part.slot, at, r), w, x, top, total);
    };
    if (b.turns == 1) {
      if (part.row0 + col <= part.last_row) {
#pragma unroll
        for (int v = 0; v < VD; v++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            const int w = 16 * v + 4 * quad + r;
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = o[v][j][r];
            if (w < b.c.W) put(head, col, w, x, run[0].m, run[0].l);
          }
      }
    } else {
#pragma unroll
      for (int v = 0; v < VD; v++)
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
          for (int j = 0; j < 8; j++)
            lds.joined.o[wave][col][128 * v + 8 * (4 * quad + r) + j] = o[v][j][r];
      if (quad == 0) {
        lds.joined.m[wave][col] = run[0].m;
        lds.joined.l[wave][col] = run[0].l;
      }
      __syncthreads();
      const int W = b.c.W;
      for (uint32_t x = threadIdx.x; x < kFewTile * held * W; x += blockDim.x) {
        const int rh = x / W, w = x - rh * W;
        uint32_t r_, hh;
        b.held.divmod(rh, r_, hh);
        const int r = r_;
        if (part.row0 + r > part.last_row) break;  // rows ascend
        float top = -INFINITY;
        for (uint32_t k = hh; k < held * b.turns; k += held) top = fmaxf(top, lds.joined.m[k][r]);
        const float ref = top == -INFINITY ? 0.0f : top;
        float total = 0, v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        for (uint32_t k = hh; k < held * b.turns; k += held) {
          const float f = __builtin_amdgcn_exp2f(lds.joined.m[k][r] - ref);
          total += f * lds.joined.l[k][r];
#pragma unroll
          for (int j = 0; j < 8; j++) v[j] += f * lds.joined.o[k][r][8 * w + j];
        }
        put(group * held + hh, r, w, v, top, total);
      }
    }
    }
    if (share.count == 0) return;
    next_tile<false>(args_now(), part, share, sq);
    if (share.count == 0) return;
    __syncthreads();  // LDS is free
  }
}

template <bool kWhole, typename T>
void launch(const AttendArgs& a, uint32_t grid, hipStream_t s) {
  const int g = a.c.NG;
  if (g <= 2)
    attend_rows<2, kWhole, T><<<grid, 64 * a.held.d * a.turns, 0, s>>>(a);
  else if (g <= 3)
    attend_rows<3, kWhole, T><<<grid, 64 * a.held.d * a.turns, 0, s>>>(a);
  else if (g <= 4)
    attend_rows<4, kWhole, T><<<grid, 64 * a.held.d * a.turns, 0, s>>>(a);
  else if (g <= 6)
    attend_rows<6, kWhole, T><<<grid, 64 * a.held.d * a.turns, 0, s>>>(a);
  else
    attend_rows<8, kWhole, T><<<grid, 64 * a.held.d * a.turns, 0, s>>>(a);
}

template <typename T>
void launch_type(const AttendArgs& a, uint32_t grid, hipStream_t s) {
  if (a.c.W % 4 == 0)
    launch<true, T>(a, grid, s);
  else
    launch<false, T>(a, grid, s);
}

}  // namespace

int attend_few(const AttendArgs& a, int type, hipStream_t s) {
  const uint32_t grid = a.few.workgroups * a.groups.d;
  if (type == EVS_BF16)
    launch_type<__bf16>(a, grid, s);
  else
    launch_type<_Float16>(a, grid, s);
  EVS_LAUNCHED("evs_fp4_attend");
  return EVS_OK;
}

}  // namespace evs
