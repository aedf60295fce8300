// Attention over full-width pages for few query rows at a time (full.hpp has the mathematics).
#include "full.hpp"

namespace evs {
namespace {

// A wave's tokens of one fetch, and the loads of them that are under way: K rows as operands as they
// lie, and of V eight tokens' chunk of VW elements, which are turned within the lane.
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

  __device__ __forceinline__ void fetch(const FullArgs& a, const uint64_t* at, int lane) {
    const int col = lane & 15, quad = lane >> 4;
#pragma unroll
    for (int g = 0; g < 2; g++) {
      const uint64_t p = at[16 * g + col];
#pragma unroll
      for (int i = 0; i < NG; i++) k[g][i] = load16(p + 16 * min(4 * i + quad, a.d / 8 - 1));
    }
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

// One workgroup: a part of the context of a tile of 16 query rows and one KV head, 64 tokens of it a
// wave in turn. Nothing passes through LDS but the tokens' addresses and the waves' results.
template <typename T, int NG>
__global__ __launch_bounds__(kFullThreads, NG > 4 ? 1 : 2) void attend_full_rows(
    FullArgs a, uint32_t prefix_items) {
  typedef Fetched<NG> Rows32;
  constexpr int VD = Rows32::VD, VW = Rows32::VW;
  constexpr int kPair = 64;  // tokens of a wave's two fetches
  struct Joined {
    float o[kFullWaves][kRowTile][16 * VW * VD + 4];
    float m[kFullWaves][kRowTile], l[kFullWaves][kRowTile];
  };
  union Shared {
    uint64_t at[kFullWaves][2][kPair];
    Joined joined;
  };
  __shared__ Shared lds;

  // which rows, which part of which context
  const bool prefix = blockIdx.x < prefix_items;
  const Contexts& c = prefix ? a.pre : a.own;
  uint32_t item = prefix ? blockIdx.x : blockIdx.x - prefix_items;
  uint32_t head, rest, who, tile;
  a.div_heads.divmod(item, rest, head);
  const uint32_t split = rest / c.tiles, place = rest - split * c.tiles;
  if (prefix) {
    if (!find_place(c.n, place,
                    [&](uint32_t g) {
                      return static_cast<uint32_t>(group_rows(a, g).rows + kRowTile - 1) / kRowTile;
                    },
                    who, tile))
      return;
  } else if (a.starts == nullptr) {
    const uint32_t per = (a.shared.d + kRowTile - 1) / kRowTile;
    who = place / per;
    tile = place - who * per;
  } else if (!find_place(c.n, place,
                         [&](uint32_t s) {
                           return static_cast<uint32_t>(sequence_rows(a, s).rows + kRowTile - 1) /
                                  kRowTile;
                         },
                         who, tile)) {
    return;
  }
  const Rows sq = scalar_rows(prefix ? group_rows(a, who) : sequence_rows(a, who));
  const int row0 = tile * kRowTile, last_row = min(row0 + kRowTile, sq.rows) - 1;
  // own tokens are seen up to the query's own, a prefix by every row
  const int past = prefix ? sq.len : sq.len - sq.nq;
  const int end = min(sq.len, past + static_cast<int>(a.shared.div(last_row)) + 1);
  const int begin = split * c.chunk;
  const int stop = static_cast<int>(split) + 1 == c.splits ? end : min(end, begin + c.chunk);
  if (begin >= stop && (prefix || split > 0)) return;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  uint32_t qi, qg;
  a.shared.divmod(min(row0 + col, last_row), qi, qg);
  const int sees = past + static_cast<int>(qi);  // this lane's row: the tokens up to this one
  const int all_see = min(stop, past + static_cast<int>(a.shared.div(row0)) + 1);
  const int32_t* table = c.tables + static_cast<int64_t>(who) * c.stride;
  const uint64_t base = reinterpret_cast<uint64_t>(a.base) + head * a.sh;

  f32x4 o[VD][VW];
#pragma unroll
  for (int v = 0; v < VD; v++)
#pragma unroll
    for (int j = 0; j < VW; j++) o[v][j] = f32x4{0, 0, 0, 0};
  Running run[1];

  const int first = begin + kPair * wave;
  if (first < stop) {
    u32x4 q[NG];
    load_query<NG>(a, a.q + (sq.q0 + qi) * a.q_token + (head * a.shared.d + qg) * a.q_head, quad,
                   q);
    const int step = kPair * kFullWaves;
    const int pairs = (stop - first + step - 1) / step;
    // (without a sign: past the last pair it may pass 2^31)
    const auto token_of = [&](int p) {
      return static_cast<uint32_t>(first) + static_cast<uint32_t>(p * step + lane);
    };
    const auto page_of = [&](int p) {
      return table[a.div_bs.div(min(token_of(p), static_cast<uint32_t>(stop) - 1))];
    };
    // the addresses of a pair's tokens, and which of them are tokens
    const auto locate = [&](int p, int32_t page) {
      const uint32_t t = token_of(p);
      uint32_t n, off;
      a.div_bs.divmod(min(t, static_cast<uint32_t>(stop) - 1), n, off);
      const bool ok = t < static_cast<uint32_t>(stop) && page >= 0 && page < a.num_blocks;
      lds.at[wave][p & 1][lane] = base + (ok ? page * a.sb + static_cast<int64_t>(off) * a.so : 0);
      return __builtin_amdgcn_ballot_w64(ok);
    };
    unsigned long long ok = locate(0, page_of(0)), ok_next = 0;
    int32_t page = page_of(1);
    Rows32 rows[2];
    rows[0].fetch(a, lds.at[wave][0], lane);
    rows[1].fetch(a, lds.at[wave][0] + 32, lane);
    for (int p = 0; p < pairs; p++) {
      ok_next = locate(p + 1, page);
      page = page_of(p + 2);
#pragma unroll
      for (int sub = 0; sub < 2; sub++) {
        Rows32& x = rows[sub];
        const int t = first + p * step + 32 * sub;
        const uint32_t there = static_cast<uint32_t>(ok >> (32 * sub));
        if (there != 0) {  // uniform
          if (32 * NG > a.d) x.trim(a, quad);
          f32x4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
          for (int i = 0; i < NG; i++)
#pragma unroll
            for (int g = 0; g < 2; g++) acc[g] = mma<T>(x.k[g][i], q[i], acc[g]);
          float s[1][8];
#pragma unroll
          for (int k = 0; k < 8; k++) s[0][k] = acc[k >> 2][k & 3];
          const bool whole = t + 32 <= all_see && there == 0xFFFFFFFFu;
          bool wild = false;
          if (!whole) {
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
            wild = t + 32 > all_see && __builtin_amdgcn_ballot_w64(wild) != 0;
          }
          float fade[1];
          if (grow<1>(s, a.scale_log2, run, fade)) {
#pragma unroll
            for (int v = 0; v < VD; v++)
#pragma unroll
              for (int j = 0; j < VW; j++) o[v][j] *= fade[0];
          }
          if (__builtin_expect(wild, false)) {
            // values that are no finite numbers are added by hand to the rows that see them
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
              for (int v = 0; v < VD; v++)
#pragma unroll
                for (int k = 0; k < VW / 2; k++) x.v[j][v][k] = tamed<T>(x.v[j][v][k]);
            const float shift = run[0].shift();
#pragma unroll 1
            for (int k = 0; k < 32; k++) {
              // the token's score is with the lanes of quarter k / 4 % 4
              float mine = s[0][0];
#pragma unroll
              for (int i = 1; i < 8; i++) mine = 4 * (k >> 4) + (k & 3) == i ? s[0][i] : mine;
              mine = __shfl(mine, col + 16 * ((k >> 2) & 3));
              if (!((there >> k) & 1) || t + k > sees) continue;
              const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(mine, a.scale_log2, -shift));
              const uint64_t row = lds.at[wave][p & 1][32 * sub + k] + a.skv;
#pragma unroll
              for (int v = 0; v < VD; v++)
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                  for (int j = 0; j < VW; j++) {
                    const int e = min(128 * v + VW * (4 * quad + r) + j, a.d - 1);
                    const uint16_t bits =
                        *reinterpret_cast<const __attribute__((address_space(1))) uint16_t*>(
                            row + 2 * e);
                    if ((bits & kWildBits<T>) == kWildBits<T>)
                      o[v][j][r] += w * static_cast<float>(__builtin_bit_cast(T, bits));
                  }
            }
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
        }
        x.fetch(a, lds.at[wave][(p + 1) & 1] + 32 * sub, lane);
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
  const int slot = prefix ? split : a.pre.splits + split;
  for (int x = threadIdx.x; x < kRowTile * words; x += kFullThreads) {
    const int r = x / words, w = x - r * words;
    if (row0 + r > last_row) break;  // rows ascend
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
    a.shared.divmod(row0 + r, i, g);
    const int token = sq.q0 + i, q_head = head * a.shared.d + g;
    if (a.joined) {
      const int64_t at = part_at(a, slot, token, q_head);
      *reinterpret_cast<f32x4*>(a.sums + at * a.d + 4 * w) = v;
      if (w == 0) {
        a.stats[2 * at] = top;
        a.stats[2 * at + 1] = total;
      }
    } else {
      finish4<T>(a, token, q_head, w, v, top, total);
    }
  }
}

template <typename T>
void launch(const FullArgs& a, uint32_t items, uint32_t prefix_items, hipStream_t s) {
  const int g = (a.d + 31) / 32;
  if (g <= 2)
    attend_full_rows<T, 2><<<items, kFullThreads, 0, s>>>(a, prefix_items);
  else if (g <= 3)
    attend_full_rows<T, 3><<<items, kFullThreads, 0, s>>>(a, prefix_items);
  else if (g <= 4)
    attend_full_rows<T, 4><<<items, kFullThreads, 0, s>>>(a, prefix_items);
  else if (g <= 6)
    attend_full_rows<T, 6><<<items, kFullThreads, 0, s>>>(a, prefix_items);
  else
    attend_full_rows<T, 8><<<items, kFullThreads, 0, s>>>(a, prefix_items);
}

}  // namespace

int full_rows(const FullArgs& a, int type, hipStream_t s) {
  const uint32_t prefix_items = a.pre.tiles * a.pre.splits * a.heads;
  const uint32_t items = prefix_items + a.own.tiles * a.own.splits * a.heads;
  if (type == EVS_BF16)
    launch<__bf16>(a, items, prefix_items, s);
  else
    launch<_Float16>(a, items, prefix_items, s);
  EVS_LAUNCHED("evs_attend");
  return EVS_OK;
}

}  // namespace evs
