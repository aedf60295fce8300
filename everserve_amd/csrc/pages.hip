// Pages of a paged cache copied inside it, and the plan that packs the used ones to its front.
#include "common.hpp"

namespace evs {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------- copying pages
constexpr int kCopyThreads = 256;
constexpr int kCopyWords = 4;  // words a thread has in flight

struct CopyArgs {
  const int64_t* layer_ptrs;
  const int32_t* src;
  const int32_t* dst;
  const int32_t* count;  // pairs in use, on the device; null: all
  uint32_t pairs;
  int32_t num_blocks;
  int64_t block_bytes;  // page stride
  uint32_t page_words;
  FastDiv div_page;
  // a page is a nest of runs of `run_words` words, outer dimensions innermost first
  FastDiv run_words;
  FastDiv extent[3];  // of the dimensions but the last
  int64_t stride[4];  // in bytes
  int dims;
};

// Word `w` of a page, from the page's first byte.
template <typename T>
__device__ __forceinline__ int64_t word_offset(const CopyArgs& a, uint32_t w) {
  if (a.dims == 0) return static_cast<int64_t>(w) * sizeof(T);
  uint32_t q, r;
  a.run_words.divmod(w, q, r);
  int64_t off = static_cast<int64_t>(r) * sizeof(T);
  for (int i = 0; i + 1 < a.dims; i++) {
    a.extent[i].divmod(q, q, r);
    off += r * a.stride[i];
  }
  return off + q * a.stride[a.dims - 1];
}

// A word of a page. The host has checked every stride and run for it, but the layers' bases are in
// device memory and may lie on any element, so it claims no alignment (the instructions are those
// of aligned words).
template <typename T>
struct Word {
  typedef T type __attribute__((aligned(1)));
};

// The words of all pairs' pages, one after another, dealt to workgroups in tiles: a tile's loads
// are issued before its first store. A pair with a page the cache does not have, or whose pages
// are one, moves nothing.
//
// Bound by memory, as a large plain copy is (4.84 TB/s): 64 pages of 64 KiB in each of 32 layers 53
// us, 5.0 TB/s; the moves of a compaction, 531 MB, 99 us, 5.4. Four words a thread keep enough
// under way for that.
template <typename T>
__global__ __launch_bounds__(kCopyThreads) void copy_pages(CopyArgs a) {
  char* base = reinterpret_cast<char*>(a.layer_ptrs[blockIdx.y]);
  uint32_t pairs = a.pairs;
  if (a.count != nullptr) {
    const int32_t c = *a.count;
    pairs = c < 0 ? 0 : min(pairs, static_cast<uint32_t>(c));
  }
  const uint64_t words = static_cast<uint64_t>(pairs) * a.page_words;  // below 2^31
  constexpr uint32_t kTile = kCopyThreads * kCopyWords;
  for (uint64_t v0 = static_cast<uint64_t>(blockIdx.x) * kTile; v0 < words;
       v0 += static_cast<uint64_t>(gridDim.x) * kTile) {
    T x[kCopyWords];
    char* to[kCopyWords];
#pragma unroll
    for (int k = 0; k < kCopyWords; k++) {
      const uint64_t v = v0 + k * kCopyThreads + threadIdx.x;
      to[k] = nullptr;
      if (v < words) {
        uint32_t pair, w;
        a.div_page.divmod(static_cast<uint32_t>(v), pair, w);
        const int32_t s = a.src[pair], d = a.dst[pair];
        if (s != d && s >= 0 && d >= 0 && s < a.num_blocks && d < a.num_blocks) {
          const int64_t off = word_offset<T>(a, w);
          x[k] = __builtin_nontemporal_load(
              reinterpret_cast<const typename Word<T>::type*>(base + s * a.block_bytes + off));
          to[k] = base + d * a.block_bytes + off;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kCopyWords; k++)
      if (to[k] != nullptr)
        __builtin_nontemporal_store(x[k], reinterpret_cast<typename Word<T>::type*>(to[k]));
  }
}

// ---------------------------------------------------------------- the plan
constexpr int kPlanThreads = 256;
constexpr int kScanThreads = 1024;

struct PlanArgs {
  const int32_t* tables;
  int64_t row_stride;
  int64_t entries;  // rows * width
  uint32_t width;
  const int32_t* counts;  // entries in use of each row; null: all
  int32_t num_blocks;
  uint32_t words;  // of the bitmap
  int32_t* tables_out;
  int32_t* src;
  int32_t* dst;
  int64_t room;
  int32_t* sizes;    // [used, moved]
  uint32_t* bitmap;  // one bit a page: in use
  uint32_t* before;  // used pages before each word of the bitmap
};

// Entry i of the tables; whether it names a page in use.
__device__ __forceinline__ bool entry(const PlanArgs& a, int64_t i, int32_t& id) {
  const int64_t row = i / a.width;
  const uint32_t col = static_cast<uint32_t>(i - row * a.width);
  id = a.tables[row * a.row_stride + col];
  const uint32_t held = a.counts == nullptr
                            ? a.width
                            : static_cast<uint32_t>(max(a.counts[row], 0));
  return col < held && id >= 0 && id < a.num_blocks;
}

__global__ __launch_bounds__(kPlanThreads) void plan_clear(PlanArgs a) {
  for (uint32_t w = blockIdx.x * kPlanThreads + threadIdx.x; w < a.words;
       w += gridDim.x * kPlanThreads)
    a.bitmap[w] = 0;
}

__global__ __launch_bounds__(kPlanThreads) void plan_mark(PlanArgs a) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * kPlanThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kPlanThreads + threadIdx.x; i < a.entries;
       i += step) {
    int32_t id;
    if (entry(a, i, id)) atomicOr(a.bitmap + (id >> 5), 1u << (id & 31));
  }
}

// Used pages before each word, by one workgroup: for more pages than fit in plan_one's LDS. All of
// the plan is bound by the latency of its launches and of its dependent loads.
__global__ __launch_bounds__(kScanThreads) void plan_scan(PlanArgs a) {
  __shared__ uint32_t s_wave[kScanThreads / 64];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t carry = 0;
  for (uint32_t w0 = 0; w0 < a.words; w0 += kScanThreads) {
    const uint32_t w = w0 + tid;
    const uint32_t c = w < a.words ? __popc(a.bitmap[w]) : 0;
    uint32_t sum = c;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t up = __shfl_up(sum, d);
      if (lane >= static_cast<uint32_t>(d)) sum += up;
    }
    if (lane == 63) s_wave[wave] = sum;
    __syncthreads();
    uint32_t base = carry, total = 0;
    for (uint32_t k = 0; k < kScanThreads / 64; k++) {
      if (k < wave) base += s_wave[k];
      total += s_wave[k];
    }
    if (w < a.words) a.before[w] = base + sum - c;
    carry += total;
    __syncthreads();
  }
  if (tid == 0) a.sizes[0] = static_cast<int32_t>(carry);
}

__device__ __forceinline__ uint32_t used_before(const PlanArgs& a, uint32_t id) {
  return a.before[id >> 5] + __popc(a.bitmap[id >> 5] & ((1u << (id & 31)) - 1));
}

// The page that is free with exactly `rank` free pages before it: bisection over the words, then
// over the word's bits.
__device__ __forceinline__ int32_t free_page(const PlanArgs& a, uint32_t rank) {
  uint32_t lo = 0, hi = a.words - 1;
  while (lo < hi) {  // the last word with at most `rank` free pages before it
    const uint32_t mid = (lo + hi + 1) >> 1;
    if (32 * mid - a.before[mid] <= rank) lo = mid; else hi = mid - 1;
  }
  uint32_t left = rank - (32 * lo - a.before[lo]);
  uint32_t bits = ~a.bitmap[lo];
  while (left-- > 0) bits &= bits - 1;
  return static_cast<int32_t>(32 * lo + __builtin_ctz(bits));
}

// The u used pages go to ids 0..u-1: those already there stay, and the others, in order, go to
// the free ids below u, in order. Every page and entry finds its place by itself from the counts.
__global__ __launch_bounds__(kPlanThreads) void plan_emit(PlanArgs a) {
  const uint32_t u = static_cast<uint32_t>(a.sizes[0]);
  // u may be num_blocks, one past the bitmap's last page
  const uint32_t stay = u < static_cast<uint32_t>(a.num_blocks) ? used_before(a, u) : u;
  const uint32_t moved = u - stay;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kPlanThreads + threadIdx.x;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kPlanThreads;
  if (first == 0) a.sizes[1] = static_cast<int32_t>(moved);
  for (int64_t id = first; id < a.num_blocks; id += step) {
    const bool used = (a.bitmap[id >> 5] >> (id & 31)) & 1;
    if (id < u && !used)
      a.dst[id - used_before(a, static_cast<uint32_t>(id))] = static_cast<int32_t>(id);
    if (id >= u && used)
      a.src[used_before(a, static_cast<uint32_t>(id)) - stay] = static_cast<int32_t>(id);
  }
  for (int64_t i = moved + first; i < a.room; i += step) a.src[i] = a.dst[i] = -1;
  for (int64_t i = first; i < a.entries; i += step) {
    int32_t id;
    if (entry(a, i, id) && static_cast<uint32_t>(id) >= u)
      id = free_page(a, used_before(a, static_cast<uint32_t>(id)) - stay);
    a.tables_out[i] = id;
  }
}

// The bitmap and its counts by one workgroup, in LDS; for small tables and caches the whole plan
// (kWhole). A launch costs about 2 us here and 3 on the host. In a graph, us a plan:
//   entries, pages     one launch   two    four
//    2,368,  2,048         6.8              11.1
//    4,096,  2,048         7.7              15.3
//    6,144,  2,048         9.5      7.7     18.3
//   13,400, 16,384        30.8     11.5     13.9
//   32,768, 16,384        51       14       20
// (random tables of 16,384 pages: 2,048 entries 9.7 in one launch, 4,096 13.6, 6,144 10.0 in two).
constexpr uint32_t kOneWords = 4096;  // 131,072 pages
constexpr int64_t kOneEntries = 1 << 15;
constexpr uint32_t kWholeWords = 512;
constexpr int64_t kWholeEntries = 1 << 12;

template <bool kWhole>
__global__ __launch_bounds__(kScanThreads) void plan_one(PlanArgs a, FastDiv width) {
  __shared__ uint32_t s_bitmap[kWhole ? kWholeWords : kOneWords];
  __shared__ uint32_t s_before[kWholeWords];
  __shared__ uint32_t s_wave[kScanThreads / 64];
  constexpr uint32_t kPer = kWhole ? 1 : kOneWords / kScanThreads;  // words a thread counts
  constexpr int kAtOnce = 4;                           // entries a thread reads at once
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t entries = static_cast<uint32_t>(a.entries);
  for (uint32_t w = tid; w < a.words; w += kScanThreads) s_bitmap[w] = 0;
  __syncthreads();
  const auto read = [&](uint32_t i0, int32_t (&id)[kAtOnce], bool (&used)[kAtOnce]) {
#pragma unroll
    for (int k = 0; k < kAtOnce; k++) {
      const uint32_t i = i0 + k * kScanThreads;
      used[k] = false;
      if (i < entries) {
        uint32_t row, col;
        width.divmod(i, row, col);
        id[k] = a.tables[row * a.row_stride + col];
        const uint32_t held = a.counts == nullptr ? a.width
                                                  : static_cast<uint32_t>(max(a.counts[row], 0));
        used[k] = col < held && id[k] >= 0 && id[k] < a.num_blocks;
      }
    }
  };
  for (uint32_t i0 = tid; i0 < entries; i0 += kAtOnce * kScanThreads) {
    int32_t id[kAtOnce];
    bool used[kAtOnce];
    read(i0, id, used);
#pragma unroll
    for (int k = 0; k < kAtOnce; k++)
      if (used[k]) atomicOr(&s_bitmap[id[k] >> 5], 1u << (id[k] & 31));
  }
  __syncthreads();
  // used pages before each word
  uint32_t count[kPer], mine = 0;
#pragma unroll
  for (uint32_t k = 0; k < kPer; k++) {
    const uint32_t w = kPer * tid + k;
    count[k] = w < a.words ? __popc(s_bitmap[w]) : 0;
    mine += count[k];
  }
  uint32_t sum = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t up = __shfl_up(sum, d);
    if (lane >= static_cast<uint32_t>(d)) sum += up;
  }
  if (lane == 63) s_wave[wave] = sum;
  __syncthreads();
  uint32_t before = sum - mine, u = 0;
  for (uint32_t k = 0; k < kScanThreads / 64; k++) {
    if (k < wave) before += s_wave[k];
    u += s_wave[k];
  }
#pragma unroll
  for (uint32_t k = 0; k < kPer; k++) {
    const uint32_t w = kPer * tid + k;
    if (w < a.words) {
      if (kWhole) {
        s_before[w] = before;
      } else {
        a.before[w] = before;
        a.bitmap[w] = s_bitmap[w];
      }
    }
    before += count[k];
  }
  if (!kWhole) {
    if (tid == 0) a.sizes[0] = static_cast<int32_t>(u);
    return;
  }
  __syncthreads();
  PlanArgs b = a;
  b.bitmap = s_bitmap;
  b.before = s_before;
  const uint32_t stay = u < static_cast<uint32_t>(a.num_blocks) ? used_before(b, u) : u;
  const uint32_t moved = u - stay;
  if (tid == 0) {
    a.sizes[0] = static_cast<int32_t>(u);
    a.sizes[1] = static_cast<int32_t>(moved);
  }
  for (uint32_t id = tid; id < static_cast<uint32_t>(a.num_blocks); id += kScanThreads) {
    const bool used = (s_bitmap[id >> 5] >> (id & 31)) & 1;
    if (used != (id >= u)) continue;
    const uint32_t at = used_before(b, id);
    if (used)
      a.src[at - stay] = static_cast<int32_t>(id);
    else
      a.dst[id - at] = static_cast<int32_t>(id);
  }
  for (int64_t i = moved + tid; i < a.room; i += kScanThreads) a.src[i] = a.dst[i] = -1;
  for (uint32_t i0 = tid; i0 < entries; i0 += kAtOnce * kScanThreads) {
    int32_t id[kAtOnce];
    bool used[kAtOnce];
    read(i0, id, used);
#pragma unroll
    for (int k = 0; k < kAtOnce; k++) {
      const uint32_t i = i0 + k * kScanThreads;
      if (i >= entries) continue;
      if (used[k] && static_cast<uint32_t>(id[k]) >= u)
        id[k] = free_page(b, used_before(b, static_cast<uint32_t>(id[k])) - stay);
      a.tables_out[i] = id[k];
    }
  }
}

uint32_t grid_of(int64_t items, int64_t most) {
  const int64_t g = (items + kPlanThreads - 1) / kPlanThreads;
  return static_cast<uint32_t>(g < 1 ? 1 : g < most ? g : most);
}

}  // namespace
}  // namespace evs

extern "C" int evs_copy_blocks(const int64_t* layer_ptrs, int64_t num_layers, const int32_t* src,
                               const int32_t* dst, int64_t num_pairs, const int32_t* count,
                               int64_t num_blocks, int64_t num_heads, int64_t head_dim,
                               int64_t block_size, const int64_t* strides, int64_t elem_size,
                               void* stream) {
  evs::clear_error();
  const char* who = "evs_copy_blocks";
  EVS_REQUIRE(strides != nullptr, "%s: a layout is five strides", who);
  EVS_REQUIRE(elem_size == 1 || elem_size == 2 || elem_size == 4, "%s: element size %lld", who,
              static_cast<long long>(elem_size));
  EVS_REQUIRE(num_layers >= 0 && num_pairs >= 0 && num_blocks >= 0 && num_heads >= 0 &&
                  head_dim >= 0 && block_size >= 0,
              "%s: negative count", who);
  EVS_REQUIRE(num_layers <= 65535, "%s: %lld layers: at most 65535 a call", who,
              static_cast<long long>(num_layers));
  EVS_REQUIRE(num_blocks < (int64_t{1} << 31), "%s: %lld pages", who,
              static_cast<long long>(num_blocks));
  if (num_layers == 0 || num_pairs == 0 || num_blocks == 0 || num_heads == 0 || head_dim == 0 ||
      block_size == 0)
    return EVS_OK;
  EVS_REQUIRE(layer_ptrs != nullptr && src != nullptr && dst != nullptr, "%s: null table", who);
  for (int i = 0; i < 5; i++)
    EVS_REQUIRE(strides[i] > 0, "%s: stride %lld", who, static_cast<long long>(strides[i]));
  EVS_REQUIRE(block_size < (int64_t{1} << 31) && num_heads < (int64_t{1} << 31) &&
                  head_dim < (int64_t{1} << 31),
              "%s: a page's dimensions", who);

  // the page's dimensions by stride, those that lie back to back as one
  struct Dim {
    int64_t extent, stride;
  } dim[4] = {{head_dim, strides[4] * elem_size},
              {block_size, strides[1] * elem_size},
              {num_heads, strides[2] * elem_size},
              {2, strides[3] * elem_size}};
  for (int i = 1; i < 4; i++)
    for (int j = i; j > 0 && dim[j].stride < dim[j - 1].stride; j--) {
      const Dim t = dim[j];
      dim[j] = dim[j - 1];
      dim[j - 1] = t;
    }
  int64_t run = elem_size;  // contiguous bytes
  int n = 0;
  Dim outer[4];
  for (const Dim& d : dim) {
    if (d.extent == 1) continue;
    if (n == 0 && d.stride == run)
      run *= d.extent;
    else if (n > 0 && d.stride == outer[n - 1].stride * outer[n - 1].extent)
      outer[n - 1].extent *= d.extent;
    else
      outer[n++] = d;
  }
  int64_t word = 16;
  const auto fits = [&](int64_t w) {
    bool ok = run % w == 0 && strides[0] * elem_size % w == 0;
    for (int i = 0; i < n; i++) ok = ok && outer[i].stride % w == 0;
    return ok;
  };
  while (word > 1 && !fits(word)) word >>= 1;

  evs::CopyArgs a{};
  int64_t words = run / word;
  for (int i = 0; i <= n; i++) {
    EVS_REQUIRE(words < (int64_t{1} << 31), "%s: a page of %lld words or more", who,
                static_cast<long long>(words));
    if (i < n) words *= outer[i].extent;
  }
  a.layer_ptrs = layer_ptrs;
  a.count = count;
  a.num_blocks = static_cast<int32_t>(num_blocks);
  a.block_bytes = strides[0] * elem_size;
  a.page_words = static_cast<uint32_t>(words);
  a.div_page = evs::FastDiv(a.page_words);
  a.run_words = evs::FastDiv(static_cast<uint32_t>(run / word));
  a.dims = n;
  for (int i = 0; i < n; i++) {
    a.stride[i] = outer[i].stride;
    if (i + 1 < n) a.extent[i] = evs::FastDiv(static_cast<uint32_t>(outer[i].extent));
  }
  // words are numbered in 31 bits: a longer list goes in several launches. With a device count the
  // first launch's pairs are the ones it may cut short, so such a list is one launch or refused.
  const int64_t most = ((int64_t{1} << 31) - 1) / words;
  EVS_REQUIRE(count == nullptr || num_pairs <= most,
              "%s: %lld pairs of pages of %lld words with a device count: at most %lld", who,
              static_cast<long long>(num_pairs), static_cast<long long>(words),
              static_cast<long long>(most));
  const hipStream_t s = evs::as_stream(stream);
  for (int64_t p = 0; p < num_pairs; p += most) {
    const int64_t m = num_pairs - p < most ? num_pairs - p : most;
    a.src = src + p;
    a.dst = dst + p;
    a.pairs = static_cast<uint32_t>(m);
    const int64_t per = evs::kCopyThreads * evs::kCopyWords;
    int64_t tiles = (m * words + per - 1) / per;
    // an unknown count may leave most tiles empty: fewer workgroups that take several
    const int64_t cap = count != nullptr ? 1 + 8192 / num_layers : 1 << 20;
    if (tiles > cap) tiles = cap;
    const dim3 grid(static_cast<uint32_t>(tiles), static_cast<uint32_t>(num_layers));
    switch (word) {
      case 16: evs::copy_pages<evs::u32x4><<<grid, evs::kCopyThreads, 0, s>>>(a); break;
      case 8: evs::copy_pages<uint64_t><<<grid, evs::kCopyThreads, 0, s>>>(a); break;
      case 4: evs::copy_pages<uint32_t><<<grid, evs::kCopyThreads, 0, s>>>(a); break;
      case 2: evs::copy_pages<uint16_t><<<grid, evs::kCopyThreads, 0, s>>>(a); break;
      default: evs::copy_pages<uint8_t><<<grid, evs::kCopyThreads, 0, s>>>(a); break;
    }
    EVS_LAUNCHED(who);
  }
  return EVS_OK;
}

extern "C" int evs_plan_compaction_workspace(int64_t num_blocks, int64_t* bytes) {
  evs::clear_error();
  EVS_REQUIRE(bytes != nullptr && num_blocks >= 0 && num_blocks < (int64_t{1} << 31),
              "evs_plan_compaction_workspace: %lld pages", static_cast<long long>(num_blocks));
  *bytes = 2 * 4 * ((num_blocks + 31) / 32);
  return EVS_OK;
}

extern "C" int evs_plan_compaction(const int32_t* tables, int64_t rows, int64_t width,
                                   int64_t row_stride, const int32_t* counts, int64_t num_blocks,
                                   int32_t* tables_out, int32_t* src, int32_t* dst, int64_t room,
                                   int32_t* sizes, void* workspace, int64_t workspace_bytes,
                                   void* stream) {
  evs::clear_error();
  const char* who = "evs_plan_compaction";
  EVS_REQUIRE(rows >= 0 && width >= 0 && width < (int64_t{1} << 31) &&
                  (width == 0 || rows <= (int64_t{1} << 40) / width),
              "%s: tables of %lld rows of %lld", who, static_cast<long long>(rows),
              static_cast<long long>(width));
  int64_t need = 0;
  if (const int rc = evs_plan_compaction_workspace(num_blocks, &need)) return rc;
  EVS_REQUIRE(sizes != nullptr && (rows * width == 0 || (tables != nullptr && tables_out != nullptr)),
              "%s: null tables or sizes", who);
  EVS_REQUIRE(room >= num_blocks / 2 && (room == 0 || (src != nullptr && dst != nullptr)),
              "%s: room for %lld moves: a cache of %lld pages may need %lld", who,
              static_cast<long long>(room), static_cast<long long>(num_blocks),
              static_cast<long long>(num_blocks / 2));
  EVS_REQUIRE(need <= workspace_bytes && (need == 0 || workspace != nullptr) &&
                  (reinterpret_cast<uintptr_t>(workspace) & 3) == 0,
              "%s: a workspace of %lld bytes, %lld needed", who,
              static_cast<long long>(workspace_bytes), static_cast<long long>(need));
  evs::PlanArgs a{};
  a.tables = tables;
  a.row_stride = row_stride;
  a.entries = rows * width;
  a.width = static_cast<uint32_t>(width > 0 ? width : 1);
  a.counts = counts;
  a.num_blocks = static_cast<int32_t>(num_blocks);
  a.words = static_cast<uint32_t>((num_blocks + 31) / 32);
  a.tables_out = tables_out;
  a.src = src;
  a.dst = dst;
  a.room = room;
  a.sizes = sizes;
  a.bitmap = static_cast<uint32_t*>(workspace);
  a.before = a.bitmap + a.words;
  const hipStream_t s = evs::as_stream(stream);
  if (a.words <= evs::kWholeWords && a.entries <= evs::kWholeEntries) {
    evs::plan_one<true><<<1, evs::kScanThreads, 0, s>>>(a, evs::FastDiv(a.width));
    EVS_LAUNCHED(who);
    return EVS_OK;
  }
  if (a.words <= evs::kOneWords && a.entries <= evs::kOneEntries) {
    evs::plan_one<false><<<1, evs::kScanThreads, 0, s>>>(a, evs::FastDiv(a.width));
    EVS_LAUNCHED(who);
  } else {
    evs::plan_clear<<<evs::grid_of(a.words, 256), evs::kPlanThreads, 0, s>>>(a);
    EVS_LAUNCHED(who);
    if (a.entries > 0) {
      evs::plan_mark<<<evs::grid_of(a.entries, 2048), evs::kPlanThreads, 0, s>>>(a);
      EVS_LAUNCHED(who);
    }
    evs::plan_scan<<<1, evs::kScanThreads, 0, s>>>(a);
    EVS_LAUNCHED(who);
  }
  const int64_t items = a.entries > num_blocks ? a.entries : num_blocks;
  evs::plan_emit<<<evs::grid_of(items, 2048), evs::kPlanThreads, 0, s>>>(a);
  EVS_LAUNCHED(who);
  return EVS_OK;
}
