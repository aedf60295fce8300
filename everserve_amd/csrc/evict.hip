// Eviction from paged caches by the weights that tokens gathered: which tokens of each layer,
// sequence and KV head stay, and their rows moved to the sequence's new pages.
#include "common.hpp"

namespace evs {
namespace {

constexpr int kRun = 8;           // tokens a thread takes side by side
constexpr uint32_t kHeld = 8192;  // masses kept in LDS
constexpr uint32_t kBins = 2048;
constexpr int kPasses = 3;
constexpr int kShift[kPasses] = {21, 10, 0};

struct ChooseArgs {
  const float* mass;  // [layers, num_blocks, heads, block_size]
  int32_t num_blocks, block_size;
  FastDiv div_bs, div_heads, div_seqs;
  const int32_t* tables;
  int64_t table_stride;
  int32_t width;
  const int32_t* lens;
  int32_t seqs, heads, budget, recent;
  int32_t* lens_out;
  int32_t* kept;  // [layers, seqs, heads, budget]
};

__device__ __forceinline__ int32_t held_tokens(int32_t len, int32_t width, int32_t block_size,
                                               int32_t num_blocks) {
  const int64_t room = static_cast<int64_t>(width) * block_size;
  len = max(len, 0);
  return num_blocks == 0 ? 0 : len > room ? static_cast<int32_t>(room) : len;
}

// Masses in order as whole numbers: -0 is 0, and what is no number comes before all others.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

typedef float f32x4 __attribute__((ext_vector_type(4)));

// The bin, from the largest down, in which `left` keys are reached, by a wave; `left` gets how many of
// the bin's keys are wanted.
__device__ __forceinline__ uint32_t reached(const uint32_t* bins, uint32_t& left) {
  const uint32_t lane = threadIdx.x & 63;
  constexpr uint32_t kOf = kBins / 64;  // a lane's bins
  const auto scan = [&](uint32_t x) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t up = __shfl_up(x, d);
      if (lane >= static_cast<uint32_t>(d)) x += up;
    }
    return x;
  };
  uint32_t mine = 0;
#pragma unroll
  for (uint32_t i = 0; i < kOf; i += 4) {
    const uint4 x = *reinterpret_cast<const uint4*>(bins + kBins - (lane + 1) * kOf + i);
    mine += x.x + x.y + x.z + x.w;
  }
  const uint32_t sum = scan(mine);
  const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(sum >= left) | (1ull << 63));
  left -= __builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(mine, l);
  // that lane's bins, one a lane
  const uint32_t top = kBins - 1 - l * kOf;
  const uint32_t one = lane < kOf ? bins[top - lane] : 0;
  const uint32_t in = scan(one);
  const int k = __builtin_ctzll(__builtin_amdgcn_ballot_w64(in >= left) | (1ull << 63));
  left -= __builtin_amdgcn_readlane(in, k) - __builtin_amdgcn_readlane(one, k);
  return top - k;
}

// One workgroup a layer, sequence and KV head. Of n tokens the `recent` last stay and the others
// with the largest masses, `budget` in all, of equal ones the first: the least mass that stays is
// found from the top bits down (11, 11 and 10 of them, by counting), then the tokens are taken in
// order. kVector: masses are read four at a time, as a page's lie.
//
// Bound by latency: its waits for memory, for LDS and for the other waves. Contexts that do not fit
// LDS are read from their pages four times, eight reads a thread under way at once. 512 of 2 to 4 Ki
// tokens 18 us; 16 of 100 to 131 Ki, a CU each, 105 us.
template <bool kVector, int kThreads>
__global__ __launch_bounds__(kThreads) void choose(ChooseArgs a) {
  constexpr int kWaves = kThreads / 64;
  constexpr int kAt = kVector ? 4 : 1;  // masses of a read
  constexpr int kAhead = 8;             // reads under way
  constexpr uint32_t kSpan = kThreads * kRun;
  __shared__ alignas(16) float s_mass[kHeld];
  __shared__ alignas(16) uint32_t s_bin[kPasses][kBins];
  __shared__ uint32_t s_wave[2][kWaves];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t head, rest, seq, layer;
  a.div_heads.divmod(blockIdx.x, rest, head);
  a.div_seqs.divmod(rest, layer, seq);
  const int32_t n = __builtin_amdgcn_readfirstlane(
      held_tokens(a.lens[seq], a.width, a.block_size, a.num_blocks));
  const int32_t stay = min(n, a.budget);
  if (layer == 0 && head == 0 && tid == 0) a.lens_out[seq] = stay;
  if (a.budget == 0) return;
  const int32_t* table = a.tables + static_cast<int64_t>(seq) * a.table_stride;
  const float* mass = a.mass + (static_cast<int64_t>(layer) * a.num_blocks * a.heads + head) *
                                   a.block_size;
  const int64_t page_stride = static_cast<int64_t>(a.heads) * a.block_size;
  int32_t* kept = a.kept + static_cast<int64_t>(blockIdx.x) * a.budget;
  const uint32_t newest = static_cast<uint32_t>(n - min(a.recent, stay));  // the first of them
  const uint32_t want = stay - (n - newest);  // others that stay
  for (int32_t j = stay + tid; j < a.budget; j += kThreads) kept[j] = -1;
  if (n <= a.budget || want == 0) {
    const uint32_t from = n <= a.budget ? 0 : newest;
    for (uint32_t j = tid; j < static_cast<uint32_t>(stay); j += kThreads) kept[j] = from + j;
    return;
  }
  const bool in_lds = newest <= kHeld;
  // A mass on a page outside the cache is less than all others; its key is 0, which no other has.
  struct Read {
    f32x4 x;
    bool there;
    __device__ uint32_t key(int i) const { return there ? key_of(x[i]) : 0; }
  };
  // kAhead reads, `step` tokens apart, from t on; past the last token they are of no page
  const auto read = [&](uint32_t t, uint32_t step, Read (&r)[kAhead]) {
    int64_t at[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; u++) {
      uint32_t p, off;
      a.div_bs.divmod(min(t + u * step, newest - 1), p, off);
      const int32_t page = table[p];
      r[u].there = page >= 0 && page < a.num_blocks;
      at[u] = r[u].there ? page * page_stride + (kVector ? off & ~3u : off) : 0;
    }
#pragma unroll
    for (int u = 0; u < kAhead; u++) {
      if constexpr (kVector)
        r[u].x = *reinterpret_cast<const f32x4*>(mass + at[u]);
      else
        r[u].x[0] = mass[at[u]];
    }
  };
  for (uint32_t b = 4 * tid; b < kPasses * kBins; b += 4 * kThreads)
    *reinterpret_cast<uint4*>(&s_bin[0][b]) = make_uint4(0, 0, 0, 0);
  __syncthreads();
  // the least key that stays, and how many of its tokens do
  uint32_t least = 0, left = want;
#pragma unroll
  for (int pass = 0; pass < kPasses; pass++) {
    const auto count = [&](uint32_t k) {
      const uint32_t above = pass == 0 ? 0 : ~uint32_t{0} << kShift[pass - 1];
      const bool in = ((k ^ least) & above) == 0;
      const uint32_t bin = (k >> kShift[pass]) & (pass == 2 ? 1023 : 2047);
      if (pass > 0) {  // few are left
        if (in) atomicAdd(&s_bin[pass][bin], 1u);
        return;
      }
      // lanes with the first lane's bin are counted at once: masses are often alike
      const uint32_t same = __builtin_amdgcn_readfirstlane(bin);
      const unsigned long long all = __builtin_amdgcn_ballot_w64(in && bin == same);
      if (in && bin != same)
        atomicAdd(&s_bin[pass][bin], 1u);
      else if (in && lane == static_cast<uint32_t>(__builtin_ctzll(all)))
        atomicAdd(&s_bin[pass][bin], static_cast<uint32_t>(__builtin_popcountll(all)));
    };
    if (pass == 0 || !in_lds) {
      for (uint32_t t0 = kAt * tid; t0 < newest; t0 += kAt * kThreads * kAhead) {
        Read r[kAhead];
        read(t0, kAt * kThreads, r);
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
          const uint32_t t = t0 + u * kAt * kThreads;
#pragma unroll
          for (int i = 0; i < kAt; i++)
            if (t + i < newest) {
              const uint32_t k = r[u].key(i);
              if (pass == 0 && in_lds) s_mass[t + i] = __builtin_bit_cast(float, k);
              count(k);
            }
        }
      }
    } else {
      for (uint32_t t = tid; t < newest; t += kThreads)
        count(__builtin_bit_cast(uint32_t, s_mass[t]));
    }
    __syncthreads();
    least |= reached(s_bin[pass], left) << kShift[pass];
  }
  uint32_t taken = 0, equal = 0;  // tokens above the least key, and with it, so far
  for (uint32_t t0 = 0, round = 0; t0 < newest; t0 += kSpan, round ^= 1) {
    const uint32_t t = t0 + kRun * tid;
    uint32_t k[kRun];
    if (in_lds) {
#pragma unroll
      for (int i = 0; i < kRun; i++)
        k[i] = t + i < newest ? __builtin_bit_cast(uint32_t, s_mass[t + i]) : 0;
    } else {
      Read r[kAhead];
      read(t, kAt, r);
#pragma unroll
      for (int i = 0; i < kRun; i++) k[i] = t + i < newest ? r[i / kAt].key(i % kAt) : 0;
    }
    uint32_t over = 0, same = 0;
#pragma unroll
    for (int i = 0; i < kRun; i++) {
      over |= (t + i < newest && k[i] > least ? 1u : 0u) << i;
      same |= (t + i < newest && k[i] == least ? 1u : 0u) << i;
    }
    // both counts of the threads before this one, 16 bits each
    const uint32_t mine = __popc(over) | __popc(same) << 16;
    uint32_t sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t up = __shfl_up(sum, d);
      if (lane >= static_cast<uint32_t>(d)) sum += up;
    }
    if (lane == 63) s_wave[round][wave] = sum;
    __syncthreads();
    uint32_t total = 0;
    sum -= mine;
    for (uint32_t w = 0; w < kWaves; w++) {
      if (w < wave) sum += s_wave[round][w];
      total += s_wave[round][w];
    }
    // of the equal ones the first `left`
    uint32_t rank = equal + (sum >> 16);
    uint32_t j = taken + (sum & 0xFFFF) + min(rank, left);
#pragma unroll
    for (int i = 0; i < kRun; i++) {
      const bool stays = (over >> i & 1) || ((same >> i & 1) && rank < left);
      rank += same >> i & 1;
      if (stays) kept[j++] = t + i;
    }
    taken += total & 0xFFFF;
    equal += total >> 16;
  }
  for (uint32_t t = newest + tid; t < static_cast<uint32_t>(n); t += kThreads)
    kept[want + (t - newest)] = t;
}

// ---------------------------------------------------------------- the rows
constexpr int kMoveThreads = 256;
constexpr int kMoveWords = 4;    // words a thread has in flight
constexpr uint32_t kPairs = 64;  // (token, head) pairs of a workgroup

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct MoveArgs {
  float* mass;
  const int64_t* layer_ptrs;
  int64_t sb, so, sh, skv;  // in bytes
  int32_t num_blocks, block_size;
  FastDiv div_bs, heads_at, words, div_seqs;  // heads of a tile; words of a half-row
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* new_tables;
  int64_t new_stride;
  int32_t new_width;
  const int32_t* lens_out;
  const int32_t* kept;
  int32_t seqs, heads, budget;
  uint32_t tokens;       // of a tile
  FastDiv token_tiles, head_tiles;
};

template <typename T>
struct MovedWord {
  typedef T type __attribute__((aligned(1)));
};

// The kept rows of a layer and sequence, in tiles of `tokens` new slots and a few heads: their
// places are worked out once into LDS, then words follow one another along a half-row, the K and
// then the V of a pair, pair by pair, and its mass. A row on a page that the cache does not have is
// not moved.
//
// Bound by the bytes: 16 layers of 4 sequences of 1,024 tokens and 8 heads of 128 105 us, 5.1 TB/s read
// and written (a large copy: 4.8). Loads and stores pass the L2 by: nothing of them is used again.
template <typename T>
__global__ __launch_bounds__(kMoveThreads) void move_kept(MoveArgs a) {
  __shared__ int64_t s_from[kPairs], s_to[kPairs];
  uint32_t rest, head_tile, token_tile, seq;
  a.head_tiles.divmod(blockIdx.x, rest, head_tile);
  a.token_tiles.divmod(rest, seq, token_tile);
  const uint32_t layer = blockIdx.y;
  const int32_t stay = a.lens_out[seq];
  const uint32_t j0 = token_tile * a.tokens;
  if (j0 >= static_cast<uint32_t>(stay)) return;
  const uint32_t tokens = min(a.tokens, stay - j0);
  const uint32_t heads = min(a.heads_at.d, a.heads - head_tile * a.heads_at.d);
  const uint32_t pairs = tokens * a.heads_at.d;  // heads past the last move nothing
  char* base = reinterpret_cast<char*>(a.layer_ptrs[layer]);
  if (threadIdx.x < pairs) {
    uint32_t token, h;
    a.heads_at.divmod(threadIdx.x, token, h);
    int64_t from = -1, to = 0;
    if (h < heads) {
      const uint32_t j = j0 + token, head = head_tile * a.heads_at.d + h;
      const int32_t t =
          a.kept[((static_cast<int64_t>(layer) * a.seqs + seq) * a.heads + head) * a.budget + j];
      uint32_t p, off, np, noff;
      a.div_bs.divmod(t, p, off);
      a.div_bs.divmod(j, np, noff);
      const int32_t page = a.tables[static_cast<int64_t>(seq) * a.table_stride + p];
      const int32_t into = static_cast<int32_t>(np) < a.new_width
                               ? a.new_tables[static_cast<int64_t>(seq) * a.new_stride + np]
                               : -1;
      if (page >= 0 && page < a.num_blocks && into >= 0 && into < a.num_blocks) {
        from = page * a.sb + static_cast<int64_t>(off) * a.so + head * a.sh;
        to = into * a.sb + static_cast<int64_t>(noff) * a.so + head * a.sh;
        float* mass = a.mass + static_cast<int64_t>(layer) * a.num_blocks * a.heads * a.block_size;
        mass[(static_cast<int64_t>(into) * a.heads + head) * a.block_size + noff] =
            mass[(static_cast<int64_t>(page) * a.heads + head) * a.block_size + off];
      }
    }
    s_from[threadIdx.x] = from;
    s_to[threadIdx.x] = to;
  }
  __syncthreads();
  const uint32_t words = pairs * 2 * a.words.d;
  for (uint32_t w0 = threadIdx.x; w0 < words; w0 += kMoveThreads * kMoveWords) {
    T x[kMoveWords];
    char* to[kMoveWords];
#pragma unroll
    for (int k = 0; k < kMoveWords; k++) {
      const uint32_t w = w0 + k * kMoveThreads;
      to[k] = nullptr;
      if (w < words) {
        uint32_t half, word;
        a.words.divmod(w, half, word);
        const int64_t from = s_from[half >> 1];
        if (from >= 0) {
          const int64_t off = (half & 1 ? a.skv : 0) + static_cast<int64_t>(word) * sizeof(T);
          x[k] = __builtin_nontemporal_load(
              reinterpret_cast<const typename MovedWord<T>::type*>(base + from + off));
          to[k] = base + s_to[half >> 1] + off;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kMoveWords; k++)
      if (to[k] != nullptr)
        __builtin_nontemporal_store(x[k], reinterpret_cast<typename MovedWord<T>::type*>(to[k]));
  }
}

}  // namespace
}  // namespace evs

extern "C" int evs_evict(const int64_t* layer_ptrs, int64_t num_layers, int64_t num_blocks,
                         int64_t num_heads, int64_t head_dim, int64_t block_size,
                         const int64_t* strides, int64_t elem_size, const int32_t* tables,
                         int64_t table_stride, int64_t width, const int32_t* lens, int64_t seqs,
                         const int32_t* new_tables, int64_t new_stride, int64_t new_width,
                         int64_t budget, int64_t recent, float* mass, int32_t* lens_out,
                         int32_t* kept, void* stream) {
  evs::clear_error();
  const char* who = "evs_evict";
  constexpr int64_t most = int64_t{1} << 31;
  EVS_REQUIRE(strides != nullptr, "%s: a layout is five strides", who);
  EVS_REQUIRE(elem_size == 1 || elem_size == 2 || elem_size == 4, "%s: element size %lld", who,
              static_cast<long long>(elem_size));
  EVS_REQUIRE(num_layers > 0 && num_layers <= 65535 && num_blocks >= 0 && num_blocks < most &&
                  num_heads > 0 && num_heads < (1 << 16) && head_dim > 0 && head_dim < (1 << 16) &&
                  block_size > 0 && block_size < most,
              "%s: bad caches: %lld layers, %lld pages, %lld heads of %lld, %lld slots a page", who,
              static_cast<long long>(num_layers), static_cast<long long>(num_blocks),
              static_cast<long long>(num_heads), static_cast<long long>(head_dim),
              static_cast<long long>(block_size));
  EVS_REQUIRE(width >= 0 && width < most && new_width >= 0 && new_width < most && seqs >= 0 &&
                  seqs < most && width * block_size < most,
              "%s: bad tables: %lld sequences, %lld and %lld pages", who,
              static_cast<long long>(seqs), static_cast<long long>(width),
              static_cast<long long>(new_width));
  EVS_REQUIRE(budget >= 0 && budget < most - 1024 && recent >= 0 && recent <= budget,
              "%s: %lld newest tokens of a budget of %lld", who, static_cast<long long>(recent),
              static_cast<long long>(budget));
  EVS_REQUIRE(new_width * block_size >= budget, "%s: %lld new pages of %lld slots hold no %lld tokens",
              who, static_cast<long long>(new_width), static_cast<long long>(block_size),
              static_cast<long long>(budget));
  EVS_REQUIRE(strides[4] == 1, "%s: a row's elements must be contiguous (element stride %lld)", who,
              static_cast<long long>(strides[4]));
  for (int i = 0; i < 4; i++)
    EVS_REQUIRE(strides[i] > 0, "%s: stride %lld", who, static_cast<long long>(strides[i]));
  if (seqs == 0) return EVS_OK;
  EVS_REQUIRE(lens != nullptr && lens_out != nullptr && (tables != nullptr || width == 0) &&
                  (new_tables != nullptr || new_width == 0) &&
                  (budget == 0 ||
                   (layer_ptrs != nullptr && mass != nullptr && kept != nullptr)),
              "%s: null argument", who);
  const int64_t items = num_layers * seqs * num_heads;
  EVS_REQUIRE(items < most / 1024, "%s: %lld layers, sequences and heads", who,
              static_cast<long long>(items));
  const hipStream_t s = evs::as_stream(stream);
  evs::ChooseArgs c{};
  c.mass = mass;
  c.num_blocks = static_cast<int32_t>(num_blocks);
  c.block_size = static_cast<int32_t>(block_size);
  c.div_bs = evs::FastDiv(static_cast<uint32_t>(block_size));
  c.div_heads = evs::FastDiv(static_cast<uint32_t>(num_heads));
  c.div_seqs = evs::FastDiv(static_cast<uint32_t>(seqs));
  c.tables = tables;
  c.table_stride = table_stride;
  c.width = static_cast<int32_t>(width);
  c.lens = lens;
  c.seqs = static_cast<int32_t>(seqs);
  c.heads = static_cast<int32_t>(num_heads);
  c.budget = static_cast<int32_t>(budget);
  c.recent = static_cast<int32_t>(recent);
  c.lens_out = lens_out;
  c.kept = kept;
  const int64_t half = head_dim * elem_size;
  int64_t word = 16;
  const auto fits = [&](int64_t w) {
    bool ok = half % w == 0;
    for (int i = 0; i < 4; i++) ok = ok && strides[i] * elem_size % w == 0;
    return ok;
  };
  while (word > 1 && !fits(word)) word >>= 1;
  evs::MoveArgs m{};
  m.layer_ptrs = layer_ptrs;
  m.sb = strides[0] * elem_size;
  m.so = strides[1] * elem_size;
  m.sh = strides[2] * elem_size;
  m.skv = strides[3] * elem_size;
  m.num_blocks = c.num_blocks;
  m.block_size = c.block_size;
  m.div_bs = c.div_bs;
  m.tables = tables;
  m.table_stride = table_stride;
  m.new_tables = new_tables;
  m.new_stride = new_stride;
  m.new_width = static_cast<int32_t>(new_width);
  m.mass = mass;
  m.lens_out = lens_out;
  m.kept = kept;
  m.seqs = c.seqs;
  m.heads = c.heads;
  m.budget = c.budget;
  const uint32_t at_once = num_heads < evs::kPairs ? static_cast<uint32_t>(num_heads) : evs::kPairs;
  m.heads_at = evs::FastDiv(at_once);
  m.head_tiles = evs::FastDiv((c.heads - 1) / at_once + 1);
  m.tokens = evs::kPairs / at_once;
  m.token_tiles = evs::FastDiv(budget > 0 ? (c.budget - 1) / m.tokens + 1 : 1);
  m.words = evs::FastDiv(static_cast<uint32_t>(half / word));
  const int64_t tiles = seqs * m.token_tiles.d * m.head_tiles.d;
  EVS_REQUIRE(tiles < most / evs::kMoveThreads, "%s: %lld tiles of rows", who,
              static_cast<long long>(tiles));
  // (a page's masses start on 16 bytes if their number is a multiple of four)
  const bool vector = block_size % 4 == 0 && reinterpret_cast<uintptr_t>(mass) % 16 == 0;
  const uint32_t grid = static_cast<uint32_t>(items);
  // twice the threads where a workgroup may have more tokens than LDS holds
  if (width * block_size > evs::kHeld) {
    if (vector)
      evs::choose<true, 1024><<<grid, 1024, 0, s>>>(c);
    else
      evs::choose<false, 1024><<<grid, 1024, 0, s>>>(c);
  } else if (vector) {
    evs::choose<true, 512><<<grid, 512, 0, s>>>(c);
  } else {
    evs::choose<false, 512><<<grid, 512, 0, s>>>(c);
  }
  EVS_LAUNCHED(who);
  if (budget == 0) return EVS_OK;
  const dim3 move(static_cast<uint32_t>(tiles), static_cast<uint32_t>(num_layers));
  switch (word) {
    case 16: evs::move_kept<evs::u32x4><<<move, evs::kMoveThreads, 0, s>>>(m); break;
    case 8: evs::move_kept<uint64_t><<<move, evs::kMoveThreads, 0, s>>>(m); break;
    case 4: evs::move_kept<uint32_t><<<move, evs::kMoveThreads, 0, s>>>(m); break;
    case 2: evs::move_kept<uint16_t><<<move, evs::kMoveThreads, 0, s>>>(m); break;
    default: evs::move_kept<uint8_t><<<move, evs::kMoveThreads, 0, s>>>(m); break;
  }
  EVS_LAUNCHED(who);
  return EVS_OK;
}
