// Attention of one new token per sequence over the paged key/value cache, the
// sequences of different lengths, several query heads to a key/value head, the
// cache in 16 or 8 bits:
//   out[b, h, :] = sum_p softmax_p(scale * Q[b, h, :] . K[p, h / group, :]) * V[p, h / group, :]
// over the positions p of sequence b below lengths[b] (with a window, the last
// `window` of them).
//
// Every visible key and value is read once and 4 * group flops are done per
// element: bound by HBM. The arithmetic still goes to the matrix cores: with
// group query heads a key element takes 2 * group multiply-adds, which at eight
// heads and 8-bit storage is more than the vector units do at the speed of the
// memory; a v_mfma_f32_16x16x32 computes 16 query columns at once (columns past
// the group idle) for a few percent of the matrix rate.
//
// A wave takes 32 keys at a time, everything in registers, no LDS:
//   S^T[key, q] = K (A operand: lane = key l % 16, 8 features per lane, straight
//                 from its row) x Q^T (B operand, fixed),
//   O^T[d, q]  += V^T (A operand: lane = feature, 8 keys per lane) x P^T (B).
// The accumulator of S^T leaves lane (q = l % 16, g = l / 16) with the keys 4g ..
// 4g+3 of either half of the tile, which is what a B operand of the second
// product holds if its contraction slots 8g .. 8g+7 are these eight keys: P^T
// is used where it is. V then wants, per lane, the same eight keys of one
// feature: a lane loads a run of consecutive features of those eight rows and
// pairs the rows up with byte permutes (32 for 8 x 8 values).
//
// The visible positions of the sequences are cut into chunks of one size, chosen on
// the device from the sum of the lengths so that there are a few for every wave that
// fits the card. A wave takes a chunk at a time and by itself: no barrier, and no wave
// waits for another's memory (with a block per chunk, its four waves meeting in LDS,
// the meeting and the start of the next chunk cost a third of the time). Every block
// works out the list of chunks (a scan over the lengths) and its waves take every n-th:
// none is empty, however the lengths are spread (a grid over sequences x chunks of
// the longest had 12000 of 16384 blocks empty at 128 sequences of 100 to 8191
// positions), and nothing but the lengths in device memory decides, so a captured
// step follows them when it is replayed. A sequence of one chunk is finished there; the
// chunks of longer ones leave partial results (maximum, sum, fp32 accumulator) that
// a second kernel joins in order. Where the cache holds short sequences only, a block
// takes a whole one instead (MEET): the second launch cost more than the meeting.

#include <algorithm>

#include "paged.hpp"

namespace oslo {
namespace {

constexpr int kTileKeys = 32;
constexpr int kColumns = 16; // query columns of a matrix product
constexpr float kLog2e = 1.4426950408889634f;
// The reference maximum of a query follows the scores when one exceeds it by more
// than this (log2 units): exponentials up to 2^8 are as exact as those up to 1.
constexpr float kRise = 8.0f;
constexpr float kLeastScore = -3.40282347e38f; // the lowest finite number

typedef float f32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Mfma16;
template <>
struct Mfma16<bf16> {
  typedef bf16 Frag __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 run(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mfma16<f16> {
  typedef f16 Frag __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 run(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

constexpr int kMinChunk = kTileKeys; // keys: one tile (by chunks, 4 sequences of 150 to 300 positions x 12 heads of 64: 8.0 us with 32, 8.6 with 64, 10.0 with 128)
constexpr int kMaxSequences = 4096; // of one launch: the chunk list of a block lies in LDS

// Chunks aimed at for `waves` waves when each of `rows` (sequences x key/value heads)
// brings one that is not full, half of one on average: one for every wave, more
// rounds where the rows alone would take most of the waves.
inline int64_t full_chunks(int64_t waves, int64_t rows) {
  return (1 + 2 * rows / waves) * waves - rows / 2;
}

struct PagedDecodeArgs {
  void *out;              // [sequences, heads, D]
  const void *q;          // [sequences, heads, D], strided
  int64_t q_seq, q_head;  // element strides
  const void *key_pages, *value_pages;
  const unsigned char *key_scales, *value_scales;
  const int *lengths;     // [sequences]
  // null: no sequence can have more than one chunk. Else the chunk list, for the join
  // ([sequences + 1] first chunks, then the chunk size), and behind it
  // [chunk][head][D + 4]: the accumulator, the maximum, the sum, two floats unused.
  int *plan;
  float *partial;
  PageMap map;
  float scale_log2e;
  int heads, group, column_groups, window;
  double full_chunks; // full_chunks() for one key/value head
};

// A word the whole wave reads, through the scalar cache. (As a vector load it would
// be waited for together with every load issued before it: the page numbers of the
// next tile would drain the keys and values in flight.)
__device__ __forceinline__ int uniform_load(const int *p) {
  return *reinterpret_cast<const __attribute__((address_space(4))) int *>(reinterpret_cast<uintptr_t>(p));
}
// The visible positions of a sequence: [first, last], empty if last < first. A
// length beyond what the sequence's table can hold is an error of the caller that
// only the device sees: `bad`, and the result is NaN.
struct Visible {
  int first, last;
  bool bad;
};
__device__ __forceinline__ Visible visible_of(const PagedDecodeArgs &a, int seq) {
  Visible v;
  int length = uniform_load(a.lengths + seq);
  const int capacity = a.map.max_pages << a.map.page_shift;
  v.bad = length > capacity;
  if (v.bad) length = capacity;
  v.last = length - 1;
  v.first = a.window > 0 && length > a.window ? length - a.window : 0;
  return v;
}

// How a lane's share of a row of V is laid out: kPer consecutive features per
// load, kLoads loads 16 * kPer features apart.
template <int D, bool E4M3>
struct ValueLayout {
  static constexpr int kPer = D == 64 ? 4 : E4M3 && D == 256 ? 16 : 8;
  static constexpr int kLoads = D / (16 * kPer);
  static constexpr int kWords = kPer * (E4M3 ? 1 : 2) / 4; // 32-bit words per load
};

template <int WORDS>
struct Words {
  uint32_t w[WORDS];
};
template <int WORDS>
__device__ __forceinline__ Words<WORDS> load_words(const char *base, uint32_t offset) {
  Words<WORDS> r;
  // (read once: the non-temporal hint; 512 MiB read at 7.0 TB/s with it, 6.0 without)
  if constexpr (WORDS == 4) {
    const u32x4_t v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(base + offset));
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = v[i];
  } else if constexpr (WORDS == 2) {
    const u32x2 v = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(base + offset));
    r.w[0] = v[0], r.w[1] = v[1];
  } else {
    r.w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t *>(base + offset));
  }
  return r;
}

// Chunks begin at the tile of the first visible position.
__device__ __forceinline__ int tiles_begin(const Visible &v) { return v.first & ~(kTileKeys - 1); }

// The list of chunks: first[s] = number of chunks of the sequences before s, first[sequences]
// that of all; returns the chunk size. An empty sequence has one chunk (which writes zeros).
__device__ __forceinline__ int list_chunks(const PagedDecodeArgs &a, int *first, float *scratch) {
  const int tid = threadIdx.x, lane = tid & (kWave - 1), n = a.map.sequences;
  auto span_of = [&](int s) __attribute__((always_inline)) -> int {
    const int length = a.lengths[s], capacity = a.map.max_pages << a.map.page_shift;
    const int end = length < 0 ? 0 : length > capacity ? capacity : length;
    const int begin = a.window > 0 && end > a.window ? end - a.window : 0;
    return end - (begin & ~(kTileKeys - 1));
  };
  auto chunk_of = [&](int64_t total) __attribute__((always_inline)) -> int {
    const double size = (double)total / a.full_chunks + 1.0;
    if (size > 1.0e9) return 1 << 30; // (no sequence is longer than 2^29)
    const int keys = ((int)size + kTileKeys - 1) / kTileKeys * kTileKeys;
    return keys < kMinChunk ? kMinChunk : keys;
  };
  auto chunks_of = [&](int span, int chunk) __attribute__((always_inline)) -> int {
    return span <= chunk ? 1 : (span + chunk - 1) / chunk;
  };
  if (n <= kWave) { // every wave by itself, a sequence per lane: all write the same list
    const int span = lane < n ? span_of(lane) : 0;
    int64_t total = span;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1)
      total += ((int64_t)__shfl_xor((int)(total >> 32), d, kWave) << 32) | (uint32_t)__shfl_xor((int)total, d, kWave);
    const int chunk = chunk_of(total);
    const int count = lane < n ? chunks_of(span, chunk) : 0;
    int upto = count;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int w = __shfl_up(upto, d, kWave);
      if (lane >= d) upto += w;
    }
    if (lane < n) first[lane] = upto - count;
    if (lane == n - 1) first[n] = upto;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    return chunk;
  }
  const int per = (n + kBlockThreads - 1) / kBlockThreads;
  int64_t *const sums = reinterpret_cast<int64_t *>(scratch); // [kWavesPerBlock]
  auto sum_over_block = [&](int64_t v, int64_t *before) __attribute__((always_inline)) -> int64_t {
    int64_t upto = v;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int64_t w = ((int64_t)__shfl_up((int)(upto >> 32), d, kWave) << 32) | (uint32_t)__shfl_up((int)upto, d, kWave);
      if (lane >= d) upto += w;
    }
    if (lane == kWave - 1) sums[tid / kWave] = upto;
    __syncthreads();
    int64_t total = 0, mine = upto - v;
#pragma unroll
    for (int w = 0; w < kWavesPerBlock; ++w) {
      if (w < tid / kWave) mine += sums[w];
      total += sums[w];
    }
    __syncthreads();
    *before = mine;
    return total;
  };
  int64_t keys = 0, before, count = 0;
  for (int i = 0; i < per; ++i)
    if (tid * per + i < n) keys += span_of(tid * per + i);
  const int chunk = chunk_of(sum_over_block(keys, &before));
  for (int i = 0; i < per; ++i)
    if (tid * per + i < n) count += chunks_of(span_of(tid * per + i), chunk);
  const int64_t all = sum_over_block(count, &before);
  for (int i = 0; i < per; ++i) {
    const int s = tid * per + i;
    if (s < n) {
      first[s] = (int)before;
      before += chunks_of(span_of(s), chunk);
    }
  }
  if (tid == 0) first[n] = (int)all;
  __syncthreads();
  return chunk;
}

// Blocks of a CU the kernel is compiled (and the grid is sized) for. (Both launches, bf16. Four at 128 features:
// 121 us instead of 94 at 131071 positions x 8 heads; six at 64: 59 instead of 40 at 8 sequences of 800 to 16000
// positions x 12 heads. In 8 bits a tile takes half the registers: four at 128 features, 189 us instead of three's 194
// at 128 sequences of 98 to 8191 positions x 8 heads, evenly spread; five spill, and three at 256 do: 351 instead of
// 202 at 128 sequences of 102 to 2048 positions x 16 heads.)
constexpr int blocks_per_cu(int D, bool e4m3) { return D == 256 ? 2 : D == 128 && !e4m3 ? 3 : 4; }

// MEET: a block per sequence and head slot, whose waves share its tiles and meet in LDS.
template <typename T, int D, bool E4M3, bool MEET>
__global__ __launch_bounds__(kBlockThreads, blocks_per_cu(D, E4M3)) void attention_paged_decode_kernel(const PagedDecodeArgs a) {
  using Op = Mfma16<T>;
  using Frag = typename Op::Frag;
  using VL = ValueLayout<D, E4M3>;
  constexpr int kElem = E4M3 ? 1 : 2;
  constexpr int kSteps = D / 32;                       // contraction steps of S^T
  constexpr int kLines = D * kElem / 128;              // 128-byte lines of a row of K (none: a line is two rows)
  constexpr int kBlocksD = D / 16;                     // 16-row blocks of O^T
  constexpr uint32_t kRowBytes = D * kElem;
  constexpr int kTurned = 8; // query columns at a time
  __shared__ __align__(16) float turn[kWavesPerBlock][kTurned][D + 4]; // a wave's own part turns its O^T
  extern __shared__ int first_chunk[]; // [sequences + 1]

  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int col = lane & 15, g = lane >> 4;

  const int chunk_keys = MEET ? 0 : list_chunks(a, first_chunk, &turn[0][0][0]);
  if (!MEET && a.plan != nullptr && blockIdx.x == 0) {
    for (int i = threadIdx.x; i <= a.map.sequences; i += kBlockThreads) a.plan[i] = first_chunk[i];
    if (threadIdx.x == 0) a.plan[a.map.sequences + 1] = chunk_keys;
  }
  const int slots = a.map.kv_heads * a.column_groups;
  const unsigned items = (unsigned)(MEET ? a.map.sequences : first_chunk[a.map.sequences]) * (unsigned)slots;

#pragma unroll 1
  for (unsigned item = blockIdx.x + (MEET ? 0u : (unsigned)wave * gridDim.x); item < items;
       item += gridDim.x * (MEET ? 1 : kWavesPerBlock)) {
  const int head_slot = (int)(item % (unsigned)slots);
  const int chunk_index = (int)(item / (unsigned)slots);
  int seq = MEET ? chunk_index : 0, chunk = 0;
  bool alone = false;
  if constexpr (!MEET) { // the last sequence whose first chunk is not behind this one
    for (int step = 1 << (31 - __builtin_clz(a.map.sequences)); step > 0; step >>= 1)
      if (seq + step < a.map.sequences && first_chunk[seq + step] <= chunk_index) seq += step;
    seq = __builtin_amdgcn_readfirstlane(seq);
    chunk = __builtin_amdgcn_readfirstlane(chunk_index - first_chunk[seq]);
    alone = __builtin_amdgcn_readfirstlane(first_chunk[seq + 1] - first_chunk[seq]) == 1;
  }
  const int kv_head = head_slot / a.column_groups;
  const int column0 = (head_slot % a.column_groups) * kColumns; // the first head of the group this block takes
  const int columns = a.group - column0 < kColumns ? a.group - column0 : kColumns;
  const int head0 = kv_head * a.group + column0;

  const Visible vis = visible_of(a, seq);
  const int begin = tiles_begin(vis);
  const int share = MEET ? ((vis.last + kTileKeys - begin) / kTileKeys + kWavesPerBlock - 1) / kWavesPerBlock * kTileKeys
                         : chunk_keys;
  const int tile0 = begin + (MEET ? wave : chunk) * share;
  const int key_end = vis.last + 1 - tile0 < share ? vis.last + 1 : tile0 + share;
  if (vis.last < vis.first) { // nothing to see
    for (int i = lane; i < columns * D; i += kWave)
      static_cast<T *>(a.out)[((int64_t)seq * a.heads + head0) * D + i] = static_cast<T>(0.f);
    continue;
  }

  // Q^T: lane (column, g) holds 8 features per step: those the lane's K operand has
  Frag qf[kSteps];
  {
    const T *qp = static_cast<const T *>(a.q) + seq * a.q_seq + (int64_t)(head0 + (col < columns ? col : 0)) * a.q_head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = kLines == 0 ? 16 * g + 8 * s : E4M3 ? 128 * (s / 4) + 32 * g + 8 * (s & 3) : 64 * (s / 2) + 16 * g + 8 * (s & 1);
      qf[s] = *reinterpret_cast<const Frag *>(qp + d);
      if (col >= columns)
#pragma unroll
        for (int i = 0; i < 8; ++i) qf[s][i] = static_cast<T>(0.f);
    }
  }

  const int *const table = a.map.table + (int64_t)seq * a.map.max_pages;
  const int page_mask = (1 << a.map.page_shift) - 1;
  const int64_t page_rows = (int64_t)a.map.kv_heads << a.map.page_shift;
  const int64_t head_rows = (int64_t)kv_head << a.map.page_shift;
  bool bad = vis.bad;

  // Rows (of the pages) at which the two halves of a tile's page slices begin.
  struct TileRows {
    int64_t row[2];
  };
  auto rows_of = [&](int key0) __attribute__((always_inline)) {
    TileRows r;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      // (a half tile wholly outside [first, last] stands on the page of the nearest visible position)
      int key = key0 + 16 * u;
      key = key > vis.last ? vis.last : key + 15 < vis.first ? vis.first : key;
      int page = uniform_load(table + (key >> a.map.page_shift));
      // A page number outside the pool must not be followed: page 0 is read in its
      // place and the result becomes NaN.
      const bool out = (unsigned)page >= (unsigned)a.map.num_pages;
      bad |= out;
      page = out ? 0 : page;
      r.row[u] = page * page_rows + head_rows;
    }
    return r;
  };
  // A lane's slot for key `key` of the tile: positions outside [first, last] read
  // a visible row instead (their probabilities are zero, and zero times a finite
  // number is zero; a row nobody has written could hold anything).
  auto slot_of = [&](int key) __attribute__((always_inline)) {
    key = key > vis.last ? vis.last : key < vis.first ? vis.first : key;
    return key;
  };

  f32x4 o[kBlocksD];
#pragma unroll
  for (int i = 0; i < kBlocksD; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f; // l: this lane's share of the sum

  // What is loaded of a tile, all before any of it is used. (Loading the next tile's keys,
  // or keys and values, while this one is computed was slower: the registers it takes cost
  // a wave per SIMD, and other waves cover the wait as well. 97, 101 and 104 us at 131071
  // positions of 8 heads x 128 in bf16.)
  Words<4> kw[2][kLines == 0 ? 1 : kLines][kLines == 0 ? 1 : 2];
  Words<VL::kWords> vw[8][VL::kLoads];
  uint32_t ks[2], vs[2];
  auto load_keys = [&](int key0, const TileRows &rows) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const char *kp = static_cast<const char *>(a.key_pages) + rows.row[u] * kRowBytes;
      if constexpr (kLines == 0) {
        const uint32_t slot = (uint32_t)(slot_of(key0 + 16 * u + col) & page_mask);
        kw[u][0][0] = load_words<4>(kp, slot * kRowBytes + 16 * g);
      } else {
        // A load takes whole lines, eight keys at a time, eight lanes to a line. (Four lanes
        // to a key, as the operand wants them, would be half a line: the load of the other
        // half finds the line pending and stalls the cache, which it did for half the
        // kernel's time.)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t slot = (uint32_t)(slot_of(key0 + 16 * u + 8 * i + (lane & 7)) & page_mask);
#pragma unroll
          for (int t = 0; t < kLines; ++t)
            kw[u][t][i] = load_words<4>(kp, slot * kRowBytes + 128 * t + 16 * (lane >> 3));
        }
      }
      if constexpr (E4M3) { // four neighbouring slots' bytes (a masked key's may be anything)
        const int at = key0 + 16 * u + 4 * g;
        ks[u] = *reinterpret_cast<const uint32_t *>(a.key_scales + rows.row[u] + (at & page_mask));
      }
    }
  };
  auto load_values = [&](int key0, const TileRows &rows) __attribute__((always_inline)) {
    if constexpr (E4M3) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
        vs[u] = *reinterpret_cast<const uint32_t *>(a.value_scales + rows.row[u] + ((key0 + 16 * u + 4 * g) & page_mask));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int u = i >> 2;
      const char *vp = static_cast<const char *>(a.value_pages) + rows.row[u] * kRowBytes;
      const uint32_t slot = (uint32_t)(slot_of(key0 + 16 * u + 4 * g + (i & 3)) & page_mask);
#pragma unroll
      for (int h = 0; h < VL::kLoads; ++h)
        vw[i][h] = load_words<VL::kWords>(vp, slot * kRowBytes + (16 * h + col) * (VL::kPer * kElem));
    }
  };
  for (int key0 = tile0; key0 < key_end; key0 += kTileKeys) {
    const bool edge = key0 < vis.first || key0 + kTileKeys > vis.last + 1; // wave-uniform
    const TileRows rows = rows_of(key0);
    load_keys(key0, rows);
    load_values(key0, rows);
    f32x4 s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      // Operands of A: lane (key l % 16, g) takes the 16-byte pieces 2 g and 2 g + 1 of its key's lines.
      // Loaded were, by lane (l % 8, b = l / 8 % 2, g), piece 2 g + b of keys l % 8 and l % 8 + 8: half the
      // lanes exchange with the lanes eight further.
      constexpr int kPieces = kLines == 0 ? 1 : 2 * kLines;
      Words<4> piece[kPieces];
      if constexpr (kLines == 0) {
        piece[0] = kw[u][0][0];
      } else {
#pragma unroll
        for (int t = 0; t < kLines; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int low = (int)kw[u][t][0].w[j], high = (int)kw[u][t][1].w[j];
            // (row_ror:8, into the upper and the lower eight lanes of every sixteen)
            piece[2 * t].w[j] = (uint32_t)__builtin_amdgcn_update_dpp(low, high, 0x128, 0xf, 0xc, false);
            piece[2 * t + 1].w[j] = (uint32_t)__builtin_amdgcn_update_dpp(high, low, 0x128, 0xf, 0x3, false);
          }
      }
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        Frag kf;
        if constexpr (E4M3) { // (the scale of the key goes onto its score)
          const Words<4> &w = piece[st / 2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const Pair<T> lo = e4m3_pair<false>(w.w[2 * (st & 1) + j], 1.0f, T());
            const Pair<T> hi = e4m3_pair<true>(w.w[2 * (st & 1) + j], 1.0f, T());
            kf[4 * j] = lo[0], kf[4 * j + 1] = lo[1], kf[4 * j + 2] = hi[0], kf[4 * j + 3] = hi[1];
          }
        } else {
          kf = __builtin_bit_cast(Frag, piece[st]);
        }
        s[u] = Op::run(kf, qf[st], s[u]);
      }
    }
    // scores in log2 units; lane (q, g): keys 4g + r of either half
    float vscale[8];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float x = s[u][r] * a.scale_log2e;
        if constexpr (E4M3) {
          x *= exponent_to_scale((int)((ks[u] >> (8 * r)) & 0xffu));
          vscale[4 * u + r] = exponent_to_scale((int)((vs[u] >> (8 * r)) & 0xffu));
        }
        if (edge) {
          const int key = key0 + 16 * u + 4 * g + r;
          const bool seen = key >= vis.first && key <= vis.last;
          x = seen ? x : -INFINITY;
          if constexpr (E4M3) vscale[4 * u + r] = seen ? vscale[4 * u + r] : 1.0f;
        }
        s[u][r] = x;
      }
    float top = s[0][0];
#pragma unroll
    for (int r = 1; r < 8; ++r) top = fmaxf(top, s[r >> 2][r & 3]);
    if (__any(top > m + kRise || m == -INFINITY)) {
      // some query's reference rises (or this is the wave's first tile)
      top = fmaxf(top, __shfl_xor(top, 16, kWave));
      top = fmaxf(top, __shfl_xor(top, 32, kWave));
      // (a finite one: keys whose scores are all -inf count as nothing, until one has a score)
      const float m_new = fmaxf(fmaxf(m, top), kLeastScore);
      const float alpha = __builtin_amdgcn_exp2f(m - m_new); // (0 in the first tile, where nothing is summed)
      l *= alpha;
#pragma unroll
      for (int i = 0; i < kBlocksD; ++i) o[i] *= alpha;
      m = m_new;
    }
    Frag p;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = __builtin_amdgcn_exp2f(s[i >> 2][i & 3] - m);
      l += e;
      p[i] = static_cast<T>(e); // (16-bit probabilities, like the prompt attention's)
    }
    // O^T: block (h, j) holds the features 16 kPer h + kPer n + j, n the row
#pragma unroll
    for (int h = 0; h < VL::kLoads; ++h) {
#pragma unroll
      for (int jj = 0; jj < VL::kPer / 2; ++jj) { // two features at a time: the pair a word of a row holds
        uint32_t pair[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (E4M3) {
            const uint32_t w = vw[i][h].w[jj / 2];
            pair[i] = __builtin_bit_cast(uint32_t, jj & 1 ? e4m3_pair<true>(w, vscale[i], T())
                                                          : e4m3_pair<false>(w, vscale[i], T()));
          } else {
            pair[i] = vw[i][h].w[jj];
          }
        }
        u32x4_t even, odd;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          even[i] = __builtin_amdgcn_perm(pair[2 * i + 1], pair[2 * i], 0x05040100u);
          odd[i] = __builtin_amdgcn_perm(pair[2 * i + 1], pair[2 * i], 0x07060302u);
        }
        const int block = VL::kPer * h + 2 * jj;
        o[block] = Op::run(__builtin_bit_cast(Frag, even), p, o[block]);
        o[block + 1] = Op::run(__builtin_bit_cast(Frag, odd), p, o[block + 1]);
      }
    }
  }

  l += __shfl_xor(l, 16, kWave);
  l += __shfl_xor(l, 32, kWave);
  if (bad) l = __builtin_nanf("");
  // O^T through the wave's LDS, to leave in rows: element r of block i is feature
  // 16 kPer (i / kPer) + kPer (4g + r) + i % kPer of query `col`
  float(*const mine)[D + 4] = turn[wave];
#pragma unroll 1
  for (int c0 = 0; c0 < columns; c0 += kTurned) {
    if constexpr (MEET) {
      __syncthreads();
    } else {
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront"); // (the rows before have been read)
      __builtin_amdgcn_wave_barrier();
    }
    if (col >= c0 && col < c0 + kTurned) {
#pragma unroll
      for (int i = 0; i < kBlocksD; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          mine[col - c0][16 * VL::kPer * (i / VL::kPer) + VL::kPer * (4 * g + r) + i % VL::kPer] = o[i][r];
      if (g == 0) mine[col - c0][D] = m, mine[col - c0][D + 1] = l;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const int rows_here = columns - c0 < kTurned ? columns - c0 : kTurned;
    if constexpr (MEET) {
      __syncthreads();
      // the waves' sums in order, relative to their common maximum (a wave without keys has -inf, and zeros)
      for (int i = threadIdx.x; i < rows_here * (D / 4); i += kBlockThreads) {
        const int c = i / (D / 4), d = 4 * (i % (D / 4));
        float top = turn[0][c][D], sum = 0.f;
#pragma unroll
        for (int w = 1; w < kWavesPerBlock; ++w) top = fmaxf(top, turn[w][c][D]);
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWavesPerBlock; ++w) {
          const float alpha = turn[w][c][D] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(turn[w][c][D] - top);
          const f32x4 v = *reinterpret_cast<const f32x4 *>(&turn[w][c][d]);
          sum = __builtin_fmaf(turn[w][c][D + 1], alpha, sum);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = __builtin_fmaf(v[e], alpha, x[e]);
        }
        typename VecOf<T, 4>::type y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = static_cast<T>(x[e] / sum);
        *reinterpret_cast<typename VecOf<T, 4>::type *>(
            static_cast<T *>(a.out) + ((int64_t)seq * a.heads + head0 + c0 + c) * D + d) = y;
      }
    } else if (alone) {
      constexpr int kRowLanes = D / 8; // lanes that store a row, eight features each
      for (int c = lane / kRowLanes; c < rows_here; c += kWave / kRowLanes) {
        const float inverse = 1.0f / mine[c][D + 1];
        typename VecOf<T, 8>::type v;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = static_cast<T>(mine[c][8 * (lane % kRowLanes) + i] * inverse);
        *reinterpret_cast<typename VecOf<T, 8>::type *>(
            static_cast<T *>(a.out) + ((int64_t)seq * a.heads + head0 + c0 + c) * D + 8 * (lane % kRowLanes)) = v;
      }
    } else {
      float *const part = a.partial + ((int64_t)chunk_index * a.heads + head0 + c0) * (D + 4);
      for (int i = lane; i < rows_here * (D / 4 + 1); i += kWave) { // (rows of D / 4 + 1 times 16 bytes)
        const int c = i / (D / 4 + 1), d = 4 * (i % (D / 4 + 1));
        *reinterpret_cast<f32x4 *>(part + (int64_t)c * (D + 4) + d) = *reinterpret_cast<const f32x4 *>(&mine[c][d]);
      }
    }
  }
  }
}

// Joins the chunks of a (sequence, head): with the common maximum M the result is
// sum_c 2^(m_c - M) o_c / sum_c 2^(m_c - M) l_c. A block per row and F features: F / 4
// threads share a chunk (four features each), the block's 1024 / F groups take every
// 1024 / F-th chunk in turn, several loads in flight, and meet in LDS; the order is
// fixed. F is 32 where there are few rows (a long sequence has hundreds of chunks, and
// more blocks read them faster: 8.2 against 12 us at 32 rows of 373), D where the rows
// fill the card by themselves.
template <typename T, int D, int kJoinFeatures>
__global__ __launch_bounds__(kBlockThreads) void attention_paged_join_kernel(const PagedDecodeArgs a) {
  constexpr int kShare = kJoinFeatures / 4, kGroups = kBlockThreads / kShare;
  __shared__ __align__(16) float sums[kGroups][kJoinFeatures + 4];
  __shared__ float group_l[kGroups], wave_m[kWavesPerBlock];
  const int row = blockIdx.x / (D / kJoinFeatures), d0 = blockIdx.x % (D / kJoinFeatures) * kJoinFeatures;
  const int tid = threadIdx.x, seq = row / a.heads;
  const int begin = uniform_load(a.plan + seq), chunks = uniform_load(a.plan + seq + 1) - begin;
  if (chunks == 1) return; // finished
  const int64_t step = (int64_t)a.heads * (D + 4); // from a chunk to the next
  const float *part = a.partial + begin * step + (int64_t)(row % a.heads) * (D + 4);
  float m = -INFINITY;
  for (int c = tid; c < chunks; c += kBlockThreads) m = fmaxf(m, part[c * step + D]);
  m = wave_allreduce(m, OpMax());
  if ((tid & (kWave - 1)) == 0) wave_m[tid / kWave] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWavesPerBlock; ++w) m = fmaxf(m, wave_m[w]);
  const int group = tid / kShare, share = tid % kShare;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
#pragma unroll 4
  for (int c = group; c < chunks; c += kGroups) {
    const float *p = part + c * step;
    const f32x4 v = *reinterpret_cast<const f32x4 *>(p + d0 + 4 * share);
    const float alpha = __builtin_amdgcn_exp2f(p[D] - m);
    l = __builtin_fmaf(p[D + 1], alpha, l);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __builtin_fmaf(v[i], alpha, x[i]);
  }
  *reinterpret_cast<f32x4 *>(&sums[group][4 * share]) = x;
  if (share == 0) group_l[group] = l;
  __syncthreads();
  if (tid < kJoinFeatures) {
    float total = 0.f, weight = 0.f;
#pragma unroll
    for (int w = 0; w < kGroups; ++w) total += sums[w][tid], weight += group_l[w];
    static_cast<T *>(a.out)[(int64_t)row * D + d0 + tid] = static_cast<T>(total / weight);
  }
}

// Where a sequence can have no more than so many tiles, a block takes it: its waves meet
// in LDS, and one launch is all. In us, against chunks and a join in brackets, bf16, one captured call after
// the other; n x L: n sequences of L / 2 to L positions, evenly spread (one of L), under a table of L:
//   64 features x 12 heads:  1 x 300 5.4 (7.7), 4 x 300 5.4 (8.1), 32 x 1024 18.2 (20.1), 400 x 1024 142 (165);
//   128 x 8, 32 query heads: 4 x 512 10.4 (9.2), 4 x 1024 17.1 (10.8), 32 x 1024 21 (25.5), 32 x 2048 37.5 (42.9);
//   256 x 16:                4 x 256 9.8 (9.9), 1 x 512 15.1 (9.0), 16 x 512 19.3 (24.1), 32 x 2048 128 (132).
// A fraction more could be gained: at 4 x 512 x 8 heads the rule takes the slower way, at 32 x 2048 too. A call that
// finds its keys in no cache waits longer: 4 sequences of up to 300 positions, 12 heads of 64, 7.6 us.
// (Asked for all sequences of a call, not for those of one of its launches: the workspace
// has to fit every launch.)
inline int64_t meet_tiles(int64_t blocks, int64_t head_dim) { return blocks >= 256 ? 32 : head_dim == 256 ? 8 : 16; }

// The grid: as many blocks as fit the card's 256 CUs at a time, or fewer where the
// sequences cannot have so many chunks. What the workspace has to hold follows from
// it: the chunk size makes at most full_chunks() chunks of all keys and heads, and
// every sequence adds one that is not full.
struct DecodeGrid {
  int64_t blocks, chunks; // chunks: at most, of one head slot
  bool join;              // some sequence may have more than one
  bool meet;              // a block takes a whole sequence
};
// `sequences` of the `all` of a call.
inline DecodeGrid decode_grid(int64_t sequences, int64_t all, int64_t kv_heads, int64_t column_groups, int64_t head_dim,
                              bool e4m3, int64_t max_length, int64_t window) {
  // (a window may begin anywhere in its first tile)
  const int64_t span = window > 0 && window < max_length ? std::min(window + kTileKeys - 1, max_length) : max_length;
  const int64_t per_sequence = std::max<int64_t>(1, (span + kMinChunk - 1) / kMinChunk);
  const int64_t slots = kv_heads * column_groups;
  DecodeGrid g;
  g.meet = per_sequence > 1 && per_sequence <= meet_tiles(all * slots, head_dim);
  if (g.meet) {
    g.blocks = sequences * slots;
    g.chunks = 0;
    g.join = false;
    return g;
  }
  // (few chunks: a block for each, so that they spread over the CUs)
  g.blocks = std::min<int64_t>(256 * blocks_per_cu((int)head_dim, e4m3), sequences * per_sequence * slots);
  g.chunks = std::min(sequences * per_sequence,
                      full_chunks(kWavesPerBlock * g.blocks, sequences * slots) / slots + 1 + sequences);
  g.join = per_sequence > 1;
  return g;
}
inline int64_t plan_ints(int64_t sequences) { return (sequences + 2 + 3) / 4 * 4; } // (whole 16 bytes)

template <typename T, int D>
int launch_paged_decode(PagedDecodeArgs a, int64_t max_length, hipStream_t stream) {
  const int64_t sequences = a.map.sequences;
  for (int64_t s0 = 0; s0 < sequences; s0 += kMaxSequences) { // (the same workspace: the stream orders them)
    PagedDecodeArgs part = a;
    const int64_t n = std::min<int64_t>(kMaxSequences, sequences - s0);
    part.map.sequences = (int)n;
    part.map.table = a.map.table + s0 * a.map.max_pages;
    part.lengths = a.lengths + s0;
    part.q = static_cast<const T *>(a.q) + s0 * a.q_seq;
    part.out = static_cast<T *>(a.out) + s0 * a.heads * D;
    const DecodeGrid grid = decode_grid(n, sequences, a.map.kv_heads, a.column_groups, D, a.key_scales != nullptr,
                                        max_length, a.window);
    const int64_t slots = (int64_t)a.map.kv_heads * a.column_groups;
    part.full_chunks = (double)full_chunks(kWavesPerBlock * grid.blocks, n * slots) / (double)slots;
    part.plan = grid.join ? reinterpret_cast<int *>(a.partial) : nullptr;
    part.partial = grid.join ? a.partial + plan_ints(n) : nullptr;
    auto *kernel = grid.meet ? (a.key_scales ? attention_paged_decode_kernel<T, D, true, true>
                                             : attention_paged_decode_kernel<T, D, false, true>)
                             : (a.key_scales ? attention_paged_decode_kernel<T, D, true, false>
                                             : attention_paged_decode_kernel<T, D, false, false>);
    const unsigned list_bytes = grid.meet ? 0u : (unsigned)((n + 1) * sizeof(int));
    kernel<<<dim3((unsigned)grid.blocks), dim3(kBlockThreads), list_bytes, stream>>>(part);
    int s = check_launch("attention_paged_decode");
    if (s != OSLO_OK) return s;
    if (!grid.join) continue;
    if (n * a.heads < 512)
      attention_paged_join_kernel<T, D, 32><<<dim3((unsigned)(n * a.heads * (D / 32))), dim3(kBlockThreads), 0, stream>>>(part);
    else
      attention_paged_join_kernel<T, D, D><<<dim3((unsigned)(n * a.heads)), dim3(kBlockThreads), 0, stream>>>(part);
    s = check_launch("attention_paged_decode(join)");
    if (s != OSLO_OK) return s;
  }
  return OSLO_OK;
}

template <typename T>
int launch_paged_decode_dim(const PagedDecodeArgs &a, int64_t head_dim, int64_t max_length, hipStream_t stream) {
  switch (head_dim) {
    case 64: return launch_paged_decode<T, 64>(a, max_length, stream);
    case 128: return launch_paged_decode<T, 128>(a, max_length, stream);
    default: return launch_paged_decode<T, 256>(a, max_length, stream);
  }
}

} // namespace
} // namespace oslo

extern "C" size_t oslo_attention_paged_decode_workspace_bytes(int64_t sequences, int64_t heads,
                                                              int64_t kv_heads, int64_t head_dim,
                                                              int64_t max_length, int64_t window) {
  using namespace oslo;
  if (sequences <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || max_length <= 0 || heads % kv_heads) return 0;
  const int64_t groups = (heads / kv_heads + kColumns - 1) / kColumns;
  const int64_t n = std::min<int64_t>(sequences, kMaxSequences); // (of one launch)
  int64_t chunks = 0; // (of either kind of cache)
  for (const bool e4m3 : {false, true}) {
    const DecodeGrid g = decode_grid(n, sequences, kv_heads, groups, head_dim, e4m3, max_length, window);
    if (!g.join) return 0;
    chunks = std::max(chunks, g.chunks);
  }
  return ((size_t)plan_ints(n) + (size_t)chunks * (size_t)heads * (size_t)(head_dim + 4)) * sizeof(float);
}

extern "C" int oslo_attention_paged_decode_fwd(void *out, const void *q, const void *key_pages,
                                               const void *value_pages, const uint8_t *key_scales,
                                               const uint8_t *value_scales, const int32_t *table,
                                               const int32_t *lengths, float *workspace, float scale,
                                               int64_t sequences, int64_t max_pages,
                                               int64_t num_pages, int64_t heads, int64_t kv_heads,
                                               int64_t page_size, int64_t head_dim, int64_t window,
                                               const int64_t *strides, int dtype,
                                               oslo_stream_t stream) {
  using namespace oslo;
  const char *const name = "oslo_attention_paged_decode_fwd";
  PagedDecodeArgs a{};
  if (heads < 0 || window < 0) return fail(OSLO_E_BAD_ARG, "%s: negative size", name);
  int s = check_pages(name, key_pages, value_pages, key_scales, value_scales, table, sequences, max_pages, num_pages,
                      kv_heads, page_size, head_dim, dtype, &a.map);
  if (s != OSLO_OK) return s;
  if (!(scale > 0.0f)) return fail(OSLO_E_BAD_ARG, "%s: the scale must be positive", name);
  if (kv_heads == 0 ? heads != 0 : heads % kv_heads != 0)
    return fail(OSLO_E_BAD_ARG, "%s: %lld query heads do not share %lld key/value heads evenly", name,
                (long long)heads, (long long)kv_heads);
  if (sequences == 0 || heads == 0) return OSLO_OK;
  if (max_pages == 0 || num_pages == 0)
    return fail(OSLO_E_BAD_ARG, "%s: a cache without pages", name);
  if (!out || !q || !lengths || !strides) return fail(OSLO_E_BAD_ARG, "%s: null pointer", name);
  if (!aligned16(out) || !aligned16(q))
    return fail(OSLO_E_UNSUPPORTED, "%s: query and output must be 16-byte aligned", name);
  if (strides[0] < 0 || strides[1] < 0 || strides[0] % 8 || strides[1] % 8)
    return fail(OSLO_E_UNSUPPORTED, "%s: strides must be multiples of 8 elements", name);
  if (heads > 8192 || sequences > (int64_t)0x7fffffff / heads) // (chunks are counted in 32 bits)
    return fail(OSLO_E_UNSUPPORTED, "%s: too many rows for one launch", name);
  const int64_t max_length = max_pages * page_size;
  a.group = (int)(heads / kv_heads);
  a.column_groups = (a.group + kColumns - 1) / kColumns;
  if (!workspace && decode_grid(std::min<int64_t>(sequences, kMaxSequences), sequences, kv_heads, a.column_groups, head_dim,
                                key_scales != nullptr, max_length, window).join)
    return fail(OSLO_E_BAD_ARG, "%s: null workspace", name);
  if (!aligned16(workspace)) return fail(OSLO_E_UNSUPPORTED, "%s: the workspace must be 16-byte aligned", name);
  a.out = out, a.q = q, a.q_seq = strides[0], a.q_head = strides[1];
  a.key_pages = key_pages, a.value_pages = value_pages, a.key_scales = key_scales, a.value_scales = value_scales;
  a.lengths = lengths;
  a.partial = workspace;
  a.scale_log2e = scale * kLog2e;
  a.heads = (int)heads;
  a.window = window >= max_length ? 0 : (int)window;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == OSLO_F16) return launch_paged_decode_dim<f16>(a, head_dim, max_length, st);
  return launch_paged_decode_dim<bf16>(a, head_dim, max_length, st);
}
