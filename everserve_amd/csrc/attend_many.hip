// Attention over 4-bit pages for sequences with many query rows: prompts and their chunks
// (attend.hpp has the mathematics).
#include "attend.hpp"

namespace evs {
namespace {

constexpr int kTile = 32;  // tokens taken at once

// One workgroup: a share of the stages of tiles of 128 query rows (64 where NG > 4) of one KV head,
// a quarter of them a wave, which all take every token of a stage. Every wave turns K's codes into
// operands for itself; V's, which take twice the instructions, are turned into operands once for
// the four waves, a quarter by each, a stage ahead, and kept in LDS in the order in which lanes
// read them.
//
// Bound by the instructions beside the products: for 32 rows and 32 tokens about 185 vector ones
// (codes to operands, exponentials, maxima, sums), and with the registers that 128 rows take a SIMD
// has two waves to fill its matrix unit from, which works 30 % of the time. The last chunks of four
// prompts (1,024 queries each of 4 to 8 Ki tokens, 32 heads on 8 of 128; 360 GFLOP, 88 MB): 505 us
// a call, 713 TFLOP/s, where a large plain bf16 product reaches 1,202 (with f16 queries 1.4 times
// as long). A whole prompt of 8,000 tokens: 1,105 us, 475 TFLOP/s (see stages_of). What carries it:
// - 128 rows a tile share the conversion of V, and two row tiles of a wave that of K (in tiles of
//   16 rows, each with its own conversions, the chunks took 811 us, in these 573);
// - the next 32 tokens' scores are under way while the weights of these are taken, across stages
//   too (564 us without, 552 with), and waves with products to issue go first (566, 548);
// - three buffers of codes, so that one barrier a stage is enough.
template <int NG, bool kWhole, typename T>
__global__ __launch_bounds__(64 * kManyWaves, 2) void attend_tiles(AttendArgs a) {
  constexpr int kTerms = QueryTerms<T>::n;
  constexpr int kRowTiles = NG > 4 ? 1 : 2;  // of 16 rows, that a wave has
  constexpr int VD = NG > 4 ? 2 : 1;      // dwords of V a lane holds of a token
  constexpr int kSubs = VD == 1 ? 2 : 1;  // 32 tokens each, of a stage
  constexpr int kTokens = kSubs * kTile;              // of a stage
  typedef Stage<NG, kTokens / kManyWaves, kManyWaves, kWhole> Rows;
  __shared__ typename Rows::Lds lds[3];
  __shared__ typename Rows::Tokens tk;
  __shared__ bf16x8 s_value[2][kSubs][VD][8][64];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Workgroups go to the 8 XCDs in turn. Each XCD gets whole heads where they divide among the
  // eight, whose rows then stay in its L2 from tile to tile; else a unit's heads go to one XCD.
  uint32_t head, owner;
  if ((a.c.heads & 7) == 0) {
    const uint32_t at = blockIdx.x >> 3, mine = static_cast<uint32_t>(a.c.heads) >> 3;
    head = (blockIdx.x & 7) * mine + at % mine;
    owner = at / mine;
  } else {
    uint32_t outer;
    a.heads.divmod(blockIdx.x >> 3, outer, head);
    owner = 8 * outer + (blockIdx.x & 7);
  }
  const char* base = a.c.base + head * a.c.sh;
  if (a.many.split && head == 0 && threadIdx.x == 0)
    a.many.tiles_in[owner] = make_uint4(0, 0, 0, 0);
  Share share;
  if (!(a.many.split || a.seqs > 64 * kManyWaves ? find_share<true>(a, owner, kTokens, share)
                                                 : longest_first(a, owner, share)))
    return;
  Sequence sq = sequence_of_all(a, share.seq);

  while (true) {
    const int lane = lane_now();
    const int col = lane & 15, quad = lane >> 4;
    const Part part = next_part<true>(a, sq, share, kTokens);
    if (part.none) return;
    if (part.slot == 1 && !part.whole && head == 0 && threadIdx.x == 0)
      describe<true>(a, share, owner, part);
    const int past = sq.len - sq.nq;
    const int row0 = part.row0, last_row = part.last_row, begin = part.begin, stop = part.stop;
    const int stages = stop > begin ? (stop - begin + kTokens - 1) / kTokens : 0;

    // this wave's rows, and the tokens that some and all of them see
    const int wave0 = row0 + 16 * kRowTiles * wave;
    const bool any_row = wave0 <= last_row;
    const int wave_last = min(wave0 + 16 * kRowTiles - 1, last_row);
    const int wave_stop =
        any_row ? min(stop, past + static_cast<int>(a.shared.div(wave_last)) + 1) : 0;
    const int all_see =
        any_row ? min(stop, past + static_cast<int>(a.shared.div(wave0)) + 1) : 0;
    int sees[kRowTiles];
    const char* qp[kRowTiles];
#pragma unroll
    for (int n = 0; n < kRowTiles; n++) {
      uint32_t qi, qg;
      a.shared.divmod(min(wave0 + 16 * n + col, last_row), qi, qg);
      sees[n] = past + static_cast<int>(qi);
      qp[n] = a.q + (sq.q0 + qi) * a.q_token + (head * a.shared.d + qg) * a.q_head;
    }

    const int32_t* table = a.tables + static_cast<int64_t>(share.seq) * a.table_stride;

    f32x4 o[kRowTiles][VD][8];
#pragma unroll
    for (int n = 0; n < kRowTiles; n++)
#pragma unroll
      for (int v = 0; v < VD; v++)
#pragma unroll
        for (int j = 0; j < 8; j++) o[n][v][j] = f32x4{0, 0, 0, 0};
    Running run[kRowTiles];

    if (stages > 0) {
      Rows rows;
      rows.place(a, wave, lane, a.one, kTokens);
      const int tid = 64 * wave + lane;
      // (without a sign: past the last stage it may pass 2^31)
      const auto token_of = [&](int stage) {
        return static_cast<uint32_t>(begin) + static_cast<uint32_t>(stage * kTokens + tid);
      };
      const auto page_of = [&](int stage) {
        return Rows::page_of(a, table, token_of(stage), stop);
      };
      const auto locate = [&](int stage, int32_t page) {
        if (64 * wave < kTokens)
          Rows::locate(a, tk, stage, base, token_of(stage), stop, page, tid, kTokens);
      };
      int32_t pages[4];
#pragma unroll
      for (int k = 0; k < 4; k++) pages[k] = page_of(k);
      int32_t page = page_of(4);
#pragma unroll
      for (int k = 0; k < 4; k++) locate(k, pages[k]);
      __syncthreads();
      Rows second = rows;
      rows.fetch(a, tk.at[0], lane);
      second.fetch(a, tk.at[1], lane);
      Query<NG, T> q[kRowTiles];
#pragma unroll
      for (int n = 0; n < kRowTiles; n++) q[n].load(a, qp[n], quad);

      // this wave's quarter of V's operands: half of the elements of a dword of 32 tokens
      const int vsub = VD == 1 ? wave >> 1 : 0, vv = VD == 1 ? 0 : wave >> 1;
      const int vw = min(16 * vv + col, a.c.W - 1);
      const auto any_wild = [&](int stage) {
        return __builtin_amdgcn_ballot_w64(tk.wild[stage & 3][lane & (kManyWaves - 1)] != 0) != 0;
      };
      const auto convert = [&](int stage, int at, bool wild) {
        Values x;
        x.load(lds[at], kTile * vsub, quad, vw);
        float sc[8];
        x.to_f32(sc);
        if (__builtin_expect(wild, false)) tame(x.codes, sc);
        auto* to = &s_value[stage & 1][vsub][vv];
        const auto pair = [&](auto c_) {
          constexpr int c = decltype(c_)::value;
          bf16x8 even, odd;
          value_pair<c>(x.codes, sc, even, odd);
          (*to)[2 * c][lane] = even;
          (*to)[2 * c + 1][lane] = odd;
        };
        if (wave & 1) {
          pair(std::integral_constant<int, 2>{});
          pair(std::integral_constant<int, 3>{});
        } else {
          pair(std::integral_constant<int, 0>{});
          pair(std::integral_constant<int, 1>{});
        }
      };
      rows.store(a, lds[0], tk, 0, wave, lane);
      second.store(a, lds[1], tk, 1, wave, lane);
      rows.fetch(a, tk.at[2], lane);
      __syncthreads();
      convert(0, 0, any_wild(0));

      // Stage i is computed with while the values of the next are converted, the rows of the one
      // after are written to LDS and those of a third are on their way: one barrier a stage. (Past
      // the last stage the last token's page is read.)
      int now = 0, ahead1 = 1, ahead2 = 2;  // where the stages' rows lie in LDS
      bool wild = false, wild_next = any_wild(0);
      f32x4 first[2][kRowTiles];
      scores<NG, kRowTiles, T>(lds[0], 0, lane, a.c.W, q, first);
      for (int i = 0; i < stages; i++) {
        __syncthreads();
        rows.store(a, lds[ahead2], tk, i + 2, wave, lane);
        locate(i + 4, page);
        page = page_of(i + 5);
        rows.fetch(a, tk.at[(i + 3) & 3], lane);
        wild = wild_next;
        wild_next = any_wild(i + 1);
        convert(i + 1, ahead1, wild_next);
        const int t0 = begin + i * kTokens;

        // 32 tokens, whose scores are in `acc`; those of the next 32 go to `after`, beside the
        // products with the values: their codes are converted while the matrix cores have these.
        const auto take = [&](int sub, f32x4 (&acc)[2][kRowTiles], int rows_after, int at_after,
                              f32x4 (&after)[2][kRowTiles]) {
          const int t = t0 + kTile * sub;
          const uint32_t ok = __builtin_amdgcn_readfirstlane(tk.ok[i & 7][sub]);
          float s[kRowTiles][8];
#pragma unroll
          for (int n = 0; n < kRowTiles; n++)
#pragma unroll
            for (int k = 0; k < 8; k++) s[n][k] = acc[k >> 2][n][k & 3];
          if (t + kTile > all_see || ok != 0xFFFFFFFFu) {
            int ahead[kRowTiles];
#pragma unroll
            for (int n = 0; n < kRowTiles; n++) ahead[n] = sees[n] - t - 4 * quad;
            mask<kRowTiles>(s, ahead, ok >> (4 * quad));
          }
          float fade[kRowTiles];
          if (grow<kRowTiles>(s, a.scale_log2, run, fade)) {
#pragma unroll
            for (int n = 0; n < kRowTiles; n++)
#pragma unroll
              for (int v = 0; v < VD; v++)
#pragma unroll
                for (int j = 0; j < 8; j++) o[n][v][j] *= fade[n];
          }
          if (__builtin_expect(wild, false)) {
#pragma unroll
            for (int v = 0; v < VD; v++)
#pragma unroll
              for (int n = 0; n < kRowTiles; n++)
                add_wild(lds[now], kTile * sub, v, a.c.W, sees[n] - t, ok, s[n],
                         a.scale_log2, run[n], o[n][v]);
          }
          u32x4 p[kRowTiles][kTerms];
#pragma unroll
          for (int v = 0; v < VD; v++) {
            // all reads are under way before the weights are computed and the first product waits
            bf16x8 x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = s_value[i & 1][sub][v][j][lane];
            __builtin_amdgcn_sched_barrier(0);
            if (v == 0) {
#pragma unroll
              for (int n = 0; n < kRowTiles; n++) weights<kTerms>(s[n], a.scale_log2, run[n], p[n]);
            }
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
              for (int n = 0; n < kRowTiles; n++)
#pragma unroll
                for (int m = 0; m < kTerms; m++)
                  o[n][v][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                      x[j], __builtin_bit_cast(bf16x8, p[n][m]), o[n][v][j], 0, 0, 0);
          }
          scores<NG, kRowTiles, T>(lds[rows_after], at_after, lane, a.c.W, q, after);
          __builtin_amdgcn_s_setprio(0);
        };
        if (t0 < wave_stop) {
          if (kSubs == 1) {
            take(0, first, ahead1, 0, first);
          } else {
            f32x4 second_half[2][kRowTiles];
            take(0, first, now, kTile, second_half);
            if (t0 + kTile < wave_stop)
              take(1, second_half, ahead1, 0, first);
          }
        }
        const int free = now;
        now = ahead1;
        ahead1 = ahead2;
        ahead2 = free;
      }
      __syncthreads();  // the rows and values have been read
    }

    {
    const int lane = lane_now();
    const int col = lane & 15, quad = lane >> 4;
    // Element 8 (4 quad + r) + j of row `col` of a tile is o[n][v][j][r].
#pragma unroll
    for (int n = 0; n < kRowTiles; n++) {
      const float l = across_rows_sum(run[n].l);
      const int row = wave0 + 16 * n + col;
      if (row > last_row) continue;
#pragma unroll
      for (int v = 0; v < VD; v++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int w = 16 * v + 4 * quad + r;
          float x[8];
#pragma unroll
          for (int j = 0; j < 8; j++) x[j] = o[n][v][j][r];
          if (w >= a.c.W) continue;
          if (part.whole)
            finish<T>(a, sq, row, head, w, x, run[n].m, l);
          else
            keep(a, part_row(a, a.many, owner, part.slot, head, row - row0), w, x, run[n].m, l);
        }
    }
    }
    if (share.count == 0) return;
    next_tile<true>(a, part, share, sq);
    if (share.count == 0) return;
    __syncthreads();  // LDS is free
  }
}

template <bool kWhole, typename T>
void launch(const AttendArgs& a, uint32_t grid, hipStream_t s) {
  const int g = a.c.NG;
  if (g <= 2)
    attend_tiles<2, kWhole, T><<<grid, 64 * kManyWaves, 0, s>>>(a);
  else if (g <= 3)
    attend_tiles<3, kWhole, T><<<grid, 64 * kManyWaves, 0, s>>>(a);
  else if (g <= 4)
    attend_tiles<4, kWhole, T><<<grid, 64 * kManyWaves, 0, s>>>(a);
  else if (g <= 6)
    attend_tiles<6, kWhole, T><<<grid, 64 * kManyWaves, 0, s>>>(a);
  else
    attend_tiles<8, kWhole, T><<<grid, 64 * kManyWaves, 0, s>>>(a);
}

template <typename T>
void launch_type(const AttendArgs& a, uint32_t grid, hipStream_t s) {
  if (a.c.W % 4 == 0)
    launch<true, T>(a, grid, s);
  else
    launch<false, T>(a, grid, s);
}

}  // namespace

int attend_many(const AttendArgs& a, int type, hipStream_t s) {
  const uint32_t grid = a.many.workgroups * static_cast<uint32_t>(a.c.heads);
  if (type == EVS_BF16)
    launch_type<__bf16>(a, grid, s);
  else
    launch_type<_Float16>(a, grid, s);
  EVS_LAUNCHED("evs_fp4_attend");
  return EVS_OK;
}

}  // namespace evs
