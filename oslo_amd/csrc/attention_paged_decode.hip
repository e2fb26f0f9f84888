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
// The positions are cut into chunks, one block of four waves each (the waves take
// every fourth tile); the waves meet in LDS; where a sequence has more than one
// chunk their partial results (maximum, sum, fp32 accumulator) are joined, in
// order, by a second kernel. Lengths are read from device memory: a step can be
// captured into a graph and replayed while they grow. Chunks a sequence does not
// reach cost an empty block.

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

struct PagedDecodeArgs {
  void *out;              // [sequences, heads, D]
  const void *q;          // [sequences, heads, D], strided
  int64_t q_seq, q_head;  // element strides
  const void *key_pages, *value_pages;
  const unsigned char *key_scales, *value_scales;
  const int *lengths;     // [sequences]
  float *partial;         // [sequences][heads][chunks][D + 2], or null: one chunk per sequence
  PageMap map;
  float scale_log2e;
  int heads, group, column_groups, chunks, chunk_keys, window;
};

// The visible positions of a sequence: [first, last], empty if last < first. A
// length beyond what the sequence's table can hold is an error of the caller that
// only the device sees: `bad`, and the result is NaN.
struct Visible {
  int first, last;
  bool bad;
};
__device__ __forceinline__ Visible visible_of(const PagedDecodeArgs &a, int seq) {
  Visible v;
  int length = __builtin_amdgcn_readfirstlane(a.lengths[seq]);
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
  if constexpr (WORDS == 4) {
    const u32x4_t v = *reinterpret_cast<const u32x4_t *>(base + offset);
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = v[i];
  } else if constexpr (WORDS == 2) {
    const u32x2 v = *reinterpret_cast<const u32x2 *>(base + offset);
    r.w[0] = v[0], r.w[1] = v[1];
  } else {
    r.w[0] = *reinterpret_cast<const uint32_t *>(base + offset);
  }
  return r;
}

template <typename T, int D, bool E4M3>
__global__ __launch_bounds__(kBlockThreads, 2) void attention_paged_decode_kernel(const PagedDecodeArgs a) {
  using Op = Mfma16<T>;
  using Frag = typename Op::Frag;
  using VL = ValueLayout<D, E4M3>;
  constexpr int kElem = E4M3 ? 1 : 2;
  constexpr int kSteps = D / 32;                       // contraction steps of S^T
  constexpr int kKeyLoads = D * kElem / 64;            // 16-byte loads per lane of a row of K (four lanes a row)
  constexpr int kBlocksD = D / 16;                     // 16-row blocks of O^T
  constexpr uint32_t kRowBytes = D * kElem;
  __shared__ float merge[2][kColumns][D + 4];
  __shared__ float merge_m[kWavesPerBlock][kColumns], merge_l[kWavesPerBlock][kColumns];

  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int col = lane & 15, g = lane >> 4;

  unsigned index = blockIdx.x;
  const int head_slot = (int)(index % (unsigned)(a.map.kv_heads * a.column_groups));
  index /= (unsigned)(a.map.kv_heads * a.column_groups);
  const int chunk = (int)(index % (unsigned)a.chunks);
  const int seq = (int)(index / (unsigned)a.chunks);
  const int kv_head = head_slot / a.column_groups;
  const int column0 = (head_slot % a.column_groups) * kColumns; // the first head of the group this block takes
  const int columns = a.group - column0 < kColumns ? a.group - column0 : kColumns;
  const int head0 = kv_head * a.group + column0;

  const Visible vis = visible_of(a, seq);
  // chunks are counted from the one the first visible position lies in
  const int key_begin = (vis.first / a.chunk_keys + chunk) * a.chunk_keys;
  const int key_end = vis.last + 1 - key_begin < a.chunk_keys ? vis.last + 1 : key_begin + a.chunk_keys;
  if (key_begin > vis.last) { // nothing to see here (the joining kernel knows; alone, the block answers)
    if (a.partial == nullptr)
      for (int i = threadIdx.x; i < columns * D; i += kBlockThreads)
        static_cast<T *>(a.out)[((int64_t)seq * a.heads + head0) * D + i] = static_cast<T>(0.f);
    return;
  }

  // Q^T: lane (column, g) holds 8 features per step: those the lane's K operand has
  Frag qf[kSteps];
  {
    const T *qp = static_cast<const T *>(a.q) + seq * a.q_seq + (int64_t)(head0 + (col < columns ? col : 0)) * a.q_head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = E4M3 ? 64 * (s / 2) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g;
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
  const int tile0 = key_begin < vis.first ? (vis.first & ~(kTileKeys - 1)) : key_begin; // chunks are whole tiles

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
      int page = __builtin_amdgcn_readfirstlane(table[key >> a.map.page_shift]);
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

  for (int key0 = tile0 + wave * kTileKeys; key0 < key_end; key0 += kWavesPerBlock * kTileKeys) {
    const TileRows rows = rows_of(key0);
    const bool edge = key0 < vis.first || key0 + kTileKeys > vis.last + 1; // wave-uniform
    Words<4> kw[2][kKeyLoads];
    Words<VL::kWords> vw[8][VL::kLoads];
    uint32_t ks[2], vs[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int page_first = key0 + 16 * u; // (in the page's coordinates below)
      const char *kp = static_cast<const char *>(a.key_pages) + rows.row[u] * kRowBytes;
      const uint32_t slot = (uint32_t)(slot_of(page_first + col) & page_mask);
#pragma unroll
      for (int j = 0; j < kKeyLoads; ++j) kw[u][j] = load_words<4>(kp, slot * kRowBytes + 64 * j + 16 * g);
      if constexpr (E4M3) {
        const int at = page_first + 4 * g; // four neighbouring slots' bytes (a masked key's may be anything)
        ks[u] = *reinterpret_cast<const uint32_t *>(a.key_scales + rows.row[u] + (at & page_mask));
        vs[u] = *reinterpret_cast<const uint32_t *>(a.value_scales + rows.row[u] + (at & page_mask));
      }
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

    f32x4 s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        Frag kf;
        if constexpr (E4M3) { // (the scale of the key goes onto its score)
          const Words<4> &w = kw[u][st / 2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const Pair<T> lo = e4m3_pair<false>(w.w[2 * (st & 1) + j], 1.0f, T());
            const Pair<T> hi = e4m3_pair<true>(w.w[2 * (st & 1) + j], 1.0f, T());
            kf[4 * j] = lo[0], kf[4 * j + 1] = lo[1], kf[4 * j + 2] = hi[0], kf[4 * j + 3] = hi[1];
          }
        } else {
          const Words<4> &w = kw[u][st];
          kf = __builtin_bit_cast(Frag, w);
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
      const float m_new = fmaxf(m, top);
      const float alpha = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
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

  // the four waves' results meet: a common maximum, the sums, the accumulators
  l += __shfl_xor(l, 16, kWave);
  l += __shfl_xor(l, 32, kWave);
  if (bad) l = __builtin_nanf("");
  if (g == 0) merge_m[wave][col] = m, merge_l[wave][col] = l;
  __syncthreads();
  float m_all = merge_m[0][col];
#pragma unroll
  for (int w = 1; w < kWavesPerBlock; ++w) m_all = fmaxf(m_all, merge_m[w][col]);
  float l_all = 0.f;
#pragma unroll
  for (int w = 0; w < kWavesPerBlock; ++w) {
    const float mw = merge_m[w][col];
    l_all += merge_l[w][col] * (mw == -INFINITY ? (merge_l[w][col] != merge_l[w][col] ? 1.0f : 0.0f)
                                                : __builtin_amdgcn_exp2f(mw - m_all));
  }
  const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_all);
  // feature of element r of block i
  auto feature = [&](int i, int r) __attribute__((always_inline)) {
    return 16 * VL::kPer * (i / VL::kPer) + VL::kPer * (4 * g + r) + i % VL::kPer;
  };
  auto put = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kBlocksD; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) merge[slot][col][feature(i, r)] = o[i][r];
  };
  auto add = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kBlocksD; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[i][r] += merge[slot][col][feature(i, r)];
  };
#pragma unroll
  for (int i = 0; i < kBlocksD; ++i) o[i] *= alpha;
  if (wave >= 2) put(wave - 2);
  __syncthreads();
  if (wave < 2) add(wave);
  __syncthreads();
  if (wave < 2) put(wave);
  if (wave == 0 && g == 0) merge_m[0][col] = m_all, merge_l[0][col] = l_all;
  __syncthreads();
  for (int i = threadIdx.x; i < columns * D; i += kBlockThreads) {
    const int c = i / D, d = i % D;
    const float x = merge[0][c][d] + merge[1][c][d];
    const int64_t row = (int64_t)seq * a.heads + head0 + c;
    if (a.partial == nullptr) {
      static_cast<T *>(a.out)[row * D + d] = static_cast<T>(x / merge_l[0][c]);
    } else {
      float *part = a.partial + (row * a.chunks + chunk) * (D + 2);
      part[2 + d] = x;
      if (d == 0) part[0] = merge_m[0][c], part[1] = merge_l[0][c];
    }
  }
}

// Joins the chunks of a (sequence, head): with the common maximum M the result is
// sum_c 2^(m_c - M) o_c / sum_c 2^(m_c - M) l_c. A thread per feature, the
// chunks in order.
template <typename T, int D>
__global__ __launch_bounds__(kBlockThreads) void attention_paged_join_kernel(const PagedDecodeArgs a, int rows) {
  constexpr int kRows = kBlockThreads / D;
  const int row = blockIdx.x * kRows + threadIdx.x / D;
  const int d = threadIdx.x % D;
  if (row >= rows) return;
  const Visible vis = visible_of(a, row / a.heads);
  const int chunks = vis.last < vis.first ? 0 : vis.last / a.chunk_keys - vis.first / a.chunk_keys + 1;
  const float *part = a.partial + (int64_t)row * a.chunks * (D + 2);
  float m = -INFINITY;
  for (int c = 0; c < chunks; ++c) m = fmaxf(m, part[c * (D + 2)]);
  float x = 0.f, l = 0.f;
  for (int c = 0; c < chunks; ++c) {
    const float *p = part + c * (D + 2);
    const float alpha = __builtin_amdgcn_exp2f(p[0] - m);
    l = __builtin_fmaf(p[1], alpha, l);
    x = __builtin_fmaf(p[2 + d], alpha, x);
  }
  static_cast<T *>(a.out)[(int64_t)row * D + d] = static_cast<T>(chunks > 0 ? x / l : 0.f);
}

// Chunks per sequence and their length.
struct ChunkPlan {
  int chunks, keys;
};
inline ChunkPlan plan_chunks(int64_t sequences, int64_t kv_heads, int64_t column_groups, int64_t max_length,
                             int64_t window) {
  const int64_t rows = std::max<int64_t>(1, sequences * kv_heads * column_groups);
  const int64_t span = window > 0 && window < max_length ? window : max_length;
  constexpr int64_t kBlock = kTileKeys * kWavesPerBlock; // keys the four waves take at a time
  const int64_t wanted = std::max<int64_t>(1, (2048 + rows - 1) / rows);
  int64_t keys = (span + wanted - 1) / wanted;
  keys = std::max<int64_t>(256, (keys + kBlock - 1) / kBlock * kBlock);
  ChunkPlan p;
  p.keys = (int)std::min<int64_t>(keys, (int64_t)1 << 30);
  p.chunks = (int)((span + p.keys - 1) / p.keys);
  if (span < max_length) p.chunks += 1; // a window may begin anywhere in its first chunk
  if (p.chunks < 1) p.chunks = 1;
  return p;
}

template <typename T, int D>
int launch_paged_decode(const PagedDecodeArgs &a, hipStream_t stream) {
  const int64_t blocks = (int64_t)a.map.sequences * a.chunks * a.map.kv_heads * a.column_groups;
  if (blocks > (int64_t)0x7fffffff)
    return fail(OSLO_E_UNSUPPORTED, "oslo_attention_paged_decode_fwd: too many blocks for one launch");
  auto *kernel = a.key_scales ? attention_paged_decode_kernel<T, D, true> : attention_paged_decode_kernel<T, D, false>;
  kernel<<<dim3((unsigned)blocks), dim3(kBlockThreads), 0, stream>>>(a);
  int s = check_launch("attention_paged_decode");
  if (s != OSLO_OK || a.partial == nullptr) return s;
  const int rows = a.map.sequences * a.heads;
  constexpr int kRows = kBlockThreads / D;
  attention_paged_join_kernel<T, D><<<dim3((unsigned)((rows + kRows - 1) / kRows)), dim3(kBlockThreads), 0, stream>>>(
      a, rows);
  return check_launch("attention_paged_decode(join)");
}

template <typename T>
int launch_paged_decode_dim(const PagedDecodeArgs &a, int64_t head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 64: return launch_paged_decode<T, 64>(a, stream);
    case 128: return launch_paged_decode<T, 128>(a, stream);
    default: return launch_paged_decode<T, 256>(a, stream);
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
  const ChunkPlan p = plan_chunks(sequences, kv_heads, groups, max_length, window);
  if (p.chunks == 1) return 0;
  return (size_t)sequences * (size_t)heads * (size_t)p.chunks * (size_t)(head_dim + 2) * sizeof(float);
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
  if (heads > 65535 || sequences > (int64_t)0x7fffffff / heads)
    return fail(OSLO_E_UNSUPPORTED, "%s: too many rows for one launch", name);
  const int64_t max_length = max_pages * page_size;
  a.group = (int)(heads / kv_heads);
  a.column_groups = (a.group + kColumns - 1) / kColumns;
  const ChunkPlan plan = plan_chunks(sequences, kv_heads, a.column_groups, max_length, window);
  if (plan.chunks > 1 && !workspace) return fail(OSLO_E_BAD_ARG, "%s: null workspace", name);
  if (!aligned16(workspace)) return fail(OSLO_E_UNSUPPORTED, "%s: the workspace must be 16-byte aligned", name);
  a.out = out, a.q = q, a.q_seq = strides[0], a.q_head = strides[1];
  a.key_pages = key_pages, a.value_pages = value_pages, a.key_scales = key_scales, a.value_scales = value_scales;
  a.lengths = lengths;
  a.partial = plan.chunks > 1 ? workspace : nullptr;
  a.scale_log2e = scale * kLog2e;
  a.heads = (int)heads;
  a.chunks = plan.chunks, a.chunk_keys = plan.keys;
  a.window = window >= max_length ? 0 : (int)window;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == OSLO_F16) return launch_paged_decode_dim<f16>(a, head_dim, st);
  return launch_paged_decode_dim<bf16>(a, head_dim, st);
}
