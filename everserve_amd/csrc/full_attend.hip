// Attention over full-width pages: its one launch (full.hpp has the mathematics, full_rows.hpp and
// full_tiles.hpp the two kinds of workgroups).
#include "full_tiles.hpp"

namespace evs {
namespace {

// Items of a launch: parts for tiles of many rows (prefixes, then chunks' contexts), then parts for
// few rows (prefixes, then own tokens). They are one launch so that the products of the first run
// beside the memory traffic of the others.
struct Items {
  uint32_t tiles, tile_prefixes, row_prefixes;
};

template <typename T, int NG, bool kWhole, int kTiles>
__global__ __launch_bounds__(kFullThreads, NG > 4 ? 1 : 2) void attend_full(FullArgs a, Items n) {
  __shared__ union {
    TilesLds<NG> tiles;
    RowsLds<NG> rows;
  } lds;
  if (blockIdx.x < n.tiles)
    tiles_part<T, NG, kWhole, kTiles>(a, lds.tiles, blockIdx.x, n.tile_prefixes);
  else
    rows_part<T, NG, kWhole, (NG > 4 ? 1 : 2)>(a, lds.rows, blockIdx.x - n.tiles, n.row_prefixes);
}

// A launch without many rows.
template <typename T, int NG, bool kWhole>
__global__ __launch_bounds__(kFullThreads, NG > 4 ? 1 : 2) void attend_full_rows(FullArgs a,
                                                                                 Items n) {
  __shared__ RowsLds<NG> lds;
  rows_part<T, NG, kWhole, 1>(a, lds, blockIdx.x, n.row_prefixes);
}

template <typename T, int NG, bool kWhole>
void launch(const FullArgs& a, uint32_t items, Items n, hipStream_t s) {
  if (n.tiles == 0)
    attend_full_rows<T, NG, kWhole><<<items, kFullThreads, 0, s>>>(a, n);
  else if (NG > 4 || a.row_tiles == 1)
    attend_full<T, NG, kWhole, 1><<<items, kFullThreads, 0, s>>>(a, n);
  else if constexpr (NG <= 4)
    attend_full<T, NG, kWhole, 2><<<items, kFullThreads, 0, s>>>(a, n);
}

template <typename T, int NG>
void launch_size(const FullArgs& a, uint32_t items, Items n, hipStream_t s) {
  if (a.d == 32 * NG)
    launch<T, NG, true>(a, items, n, s);
  else
    launch<T, NG, false>(a, items, n, s);
}

template <typename T>
void launch_type(const FullArgs& a, uint32_t items, Items n, hipStream_t s) {
  const int g = (a.d + 31) / 32;
  if (g <= 2)
    launch_size<T, 2>(a, items, n, s);
  else if (g <= 3)
    launch_size<T, 3>(a, items, n, s);
  else if (g <= 4)
    launch_size<T, 4>(a, items, n, s);
  else if (g <= 6)
    launch_size<T, 6>(a, items, n, s);
  else
    launch_size<T, 8>(a, items, n, s);
}

}  // namespace

int full_attend(const FullArgs& a, int type, hipStream_t s) {
  // tiles of one head and part are dealt to one XCD: units of them in eights
  const auto in_eights = [&](const Cut& c) {
    return (static_cast<uint32_t>(c.splits) * a.heads + 7) / 8 * 8 * c.tiles;
  };
  const uint32_t prefixes = a.group.tiles * a.group.splits * a.heads;
  Items n{};
  n.tile_prefixes = a.few_groups ? 0 : in_eights(a.group);
  n.tiles = n.tile_prefixes + in_eights(a.many);
  n.row_prefixes = a.few_groups ? prefixes : 0;
  const uint32_t items = n.tiles + n.row_prefixes + a.few.tiles * a.few.splits * a.heads;
  if (items == 0) return EVS_OK;
  if (type == EVS_BF16)
    launch_type<__bf16>(a, items, n, s);
  else
    launch_type<_Float16>(a, items, n, s);
  EVS_LAUNCHED("evs_attend");
  return EVS_OK;
}

}  // namespace evs
