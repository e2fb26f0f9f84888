// Launches of the prompt attention's backward over [batch, head, position]
// tensors (the kernel that recomputes the scores: attention_prefill_bwd.hpp),
// the pass that reads the tile store, and the entry points.

#include <algorithm>

#include "attention_prefill_bwd.hpp"

namespace oslo {
namespace {

template <typename T, int D, int ROLE, bool STORE = false>
int launch_role(const BwdArgs &a, hipStream_t stream) {
  const dim3 grid((unsigned)(8 * a.head_groups * a.own_blocks));
  constexpr unsigned kLds = sched_lds_bytes<T, D, ROLE>();
  auto go = [&]<bool HAS_PAD, bool DROP>() -> int {
    auto *kernel = a.window > 0 ? attention_bwd_kernel<T, D, ROLE, HAS_PAD, true, DROP, STORE>
                                : attention_bwd_kernel<T, D, ROLE, HAS_PAD, false, DROP, STORE>;
    if (kLds > 64u * 1024u) {
      const int s = raise_lds_limit(reinterpret_cast<const void *>(kernel), kLds, "oslo_attention_prefill_bwd");
      if (s != OSLO_OK) return s;
    }
    kernel<<<grid, dim3(kBlockThreads), kLds, stream>>>(a);
    return check_launch("attention_prefill_bwd");
  };
  if (a.pad != nullptr) {
    if (a.drop.drop) return go.template operator()<true, true>();
    return go.template operator()<true, false>();
  }
  if (a.drop.drop) return go.template operator()<false, true>();
  return go.template operator()<false, false>();
}

// dK and dV from the tile store: dK^T += Q^T dS and dV^T += dO^T P over the query
// tiles from the diagonal on, nothing else: no scores, no exponentials, no
// mask, no dropout (all of it is in the stored tiles). A block owns 32 keys per
// wave (256 with eight waves) and one of the two gradients (even blocks dK, odd
// blocks dV); a pair of waves has 64 keys and each wave of the pair half of the
// features, so a wave holds one accumulator of 64 keys x D / 2 features (D / 2
// registers), no fixed operands, and uses every transposed operand of Q (or
// dO) it reads from LDS for two products. The tiles of Q (or dO) go through LDS
// as in the other passes (three buffers: tile t is read while t + 1 and t + 2
// are on their way), shared by the block; every wave loads one 2 KiB tile of dS
// (or P) beside them, which it and its partner read back transposed, key slot
// in the lane: lane c holds the key at slot c of the store's rows, key c with
// bits 2 and 3 swapped. What this pass waits for is its loads (with none of
// them issued it takes 0.22 ms instead of 0.40 at [8,16,2048,256], without its
// products still 0.39): the more keys share a tile of Q, the fewer bytes per
// product, hence eight waves.
// Tiles of a tensor in LDS: the one that is read and those on their way. (The
// pass is bound by its loads, but not by their latency: with four or five
// buffers at 256 features, 128 and 160 KiB, it takes the same time as with three.
// Nor does it help to issue the loads of half of the waves one operand later
// than those of the others: 430 against 390 us.)
#ifndef OSLO_STORED_BUFFERS
#define OSLO_STORED_BUFFERS 3
#endif
constexpr int stored_buffers(int D) { return D == 256 ? OSLO_STORED_BUFFERS : 3; }
// waves of a block (32 keys each), by head size
constexpr int stored_waves(int D) { return D == 64 ? 4 : OSLO_STORED_WAVES; }

template <typename T, int D>
constexpr unsigned stored_lds_bytes() {
  return (unsigned)stored_buffers(D) * (kSchedTile * D * sizeof(T) + stored_waves(D) * kStoredTileBytes);
}

// blocks that share a CU: what the 160 KiB of LDS hold, four at most
template <typename T, int D>
constexpr int stored_blocks_per_cu() {
  const unsigned fit = 160u * 1024u / stored_lds_bytes<T, D>();
  return fit > 4u ? 4 : (int)fit;
}

template <typename T, int D, bool HAS_WINDOW>
__global__ __launch_bounds__(stored_waves(D) * kWave, (stored_blocks_per_cu<T, D>())) void attention_bwd_stored_kernel(
    const BwdArgs a) {
  constexpr int kStoredWaves = stored_waves(D);
  constexpr int kStoredKeys = 32 * kStoredWaves; // keys of a block
  constexpr int kStoredBuffers = stored_buffers(D);
  using Op = MatrixOp<T>;
  using Frag = typename Op::Frag;
  constexpr int kChunks = D / 8;
  constexpr int kBlocksD = D / 32;
  constexpr int kTile = kSchedTile * D;
  constexpr int kRowBytes = D * (int)sizeof(T);
  constexpr int kSwizzle = kChunks >= 16 ? 15 : 7;
  constexpr int kLoadsN = kSchedTile * kChunks / (kStoredWaves * kWave); // loads per thread and tile of Q (or dO)
  static_assert(kLoadsN >= 1, "a tile of fewer entries than the block has threads");
  constexpr int kItems = kLoadsN + 2;  // and the wave's own tile of the store
  constexpr int kHalfBlocks = kBlocksD / 2; // 32-feature blocks of a wave's half of the features
  constexpr int kOperands = 2 * kHalfBlocks; // transposed operands of Q or dO per tile, each used for both key tiles

  extern __shared__ __align__(1024) unsigned char lds_raw[];
  T *const t_lds = reinterpret_cast<T *>(lds_raw); // [3][query][chunk ^ f(query)][8]

  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int half = lane >> 5;
  const int col = lane & 31;
  // two pairs of waves, 64 keys each; of a pair, a wave per half of the features
  const int feature_half = wave & 1;
  unsigned char *const x_lds = reinterpret_cast<unsigned char *>(t_lds + kStoredBuffers * kTile) +
                               wave * (kStoredBuffers * kStoredTileBytes); // [3][query][slot]
  // the two stored tiles the wave multiplies with: its own and its partner's
  const unsigned char *const x_pair = reinterpret_cast<unsigned char *>(t_lds + kStoredBuffers * kTile) +
                                      (wave & ~1) * (kStoredBuffers * kStoredTileBytes);

  const int xcd = blockIdx.x & 7;
  const int slot = blockIdx.x >> 4;
  const bool for_dv = ((blockIdx.x >> 3) & 1) != 0;
  // The blocks of a head follow one another on one XCD, the longest walk
  // first: the two or three heads an XCD works on at a time keep their Q and dO
  // (2 x S x D values each) in its L2 while every block of the head reads them.
  const int S = a.S;
  const int key_blocks = (S + kStoredKeys - 1) / kStoredKeys;
  const int bh = a.bh0 + xcd + 8 * (slot / key_blocks);
  const int own_block = slot % key_blocks;
  if (bh >= a.batch_heads) return; // the whole block
  const int b = bh / a.heads;
  const int hd = bh - b * a.heads;
  const int own0 = own_block * kStoredKeys;
  const int key_tile = own0 / 32 + wave; // the key tile whose stored tiles this wave loads
  const int window = HAS_WINDOW ? a.window : 0;

  const int first_tile = own0 / kSchedTile;
  int last_query = S - 1;
  if (HAS_WINDOW && own0 + kStoredKeys - 1 + window - 1 < last_query) last_query = own0 + kStoredKeys - 1 + window - 1;
  const int tiles = last_query / kSchedTile + 1;

  const Strides3 &st_in = for_dv ? a.sdo : a.sq;
  const T *in_p = static_cast<const T *>(for_dv ? a.dout : a.q) + b * st_in.b + hd * st_in.h;
  const uint32_t in_row = (uint32_t)st_in.s * sizeof(T);
  // The permutation of a row's 16-byte chunks in LDS: chunk c of row r lies at
  // c ^ f(r). A transposing read takes, per half of the wave, 4 chunks (64 bytes)
  // of 4 consecutive rows, and rows lie a multiple of 256 bytes apart: with the
  // rows' low two bits in bits 2 and 3 of f the four rows use four different
  // quarters of the banks. (The permutation of the other passes, which leaves two
  // rows on the same banks, costs every such read two cycles.)
  constexpr bool kQuads = kChunks >= 16;
  auto f_of = [](int r) __attribute__((always_inline)) {
    if (kQuads) return ((r & 3) << 2) | ((r >> 2) & 3);
    return (((r & 3) << 1) | ((r >> 2) & 1) | (r & 8)) & kSwizzle;
  };
  // load j of a thread: entry (kStoredWaves j + wave) * 64 + lane of the tile
  uint32_t src_off[kLoadsN];
#pragma unroll
  for (int j = 0; j < kLoadsN; ++j) {
    const int entry = (kStoredWaves * j + wave) * kWave + lane;
    const int row = entry / kChunks, at = entry % kChunks;
    src_off[j] = (uint32_t)row * in_row + (uint32_t)(at ^ f_of(row)) * 16u;
  }
  TileStream src; // the next tile to load
  src.start(in_p, (uint32_t)(((int64_t)(S - 1) * st_in.s + D) * sizeof(T)), in_row, kSchedTile, first_tile, tiles);
  // The wave's tile of the store for query tile qt: nothing (zeros, without a
  // memory access) where the pass that writes the store left none: above the
  // diagonal, past the last query tile, and before the first key tile that the
  // block owning qt walks under a window.
  uint64_t store_at = reinterpret_cast<uint64_t>(a.tiles) +
                      (uint64_t)(((int64_t)(bh - a.bh0) * a.head_tiles + (int64_t)first_tile * (first_tile + 1) / 2 + key_tile) *
                                     kStoredPairBytes +
                                 (for_dv ? 0 : kStoredTileBytes));
  int store_tile = first_tile; // the query tile store_at belongs to
  auto store_descriptor = [&]() __attribute__((always_inline)) {
    bool there = store_tile >= key_tile && store_tile < tiles;
    if constexpr (HAS_WINDOW) {
      const int walk0 = (store_tile / 4) * kOwnPerBlock - window + 1;
      there = there && key_tile >= (walk0 > 0 ? walk0 / kSchedTile : 0);
    }
    u32x4 d;
    d[0] = __builtin_amdgcn_readfirstlane((uint32_t)store_at);
    d[1] = __builtin_amdgcn_readfirstlane((uint32_t)(store_at >> 32) & 0xffffu);
    d[2] = __builtin_amdgcn_readfirstlane(there ? (uint32_t)kStoredTileBytes : 0u);
    d[3] = 0x00020000u;
    return d;
  };
  int t = first_tile;
  int buf_now = 0, buf_load = 0; // buffers of tile t and of the tile being loaded (t + kStoredBuffers - 1 in the loop)
  auto next_buffer = [](int b) __attribute__((always_inline)) { return b == kStoredBuffers - 1 ? 0 : b + 1; };
  // item `it` of the loads of the next tile to load
  auto stage_item = [&](int it) __attribute__((always_inline)) {
    if (it < kLoadsN) {
      lds_load_b128(src.descriptor(), t_lds + buf_load * kTile + (kStoredWaves * it + wave) * (kWave * 8), src_off[it]);
      if (it == kLoadsN - 1) src.advance();
      return;
    }
    it -= kLoadsN;
    // (read once: past the caches' usual replacement, so that the tiles of Q and dO stay)
    // LDS gets rows of [query][slot] (lane L of load `it`: query 16 it + L / 4, 16-byte chunk L % 4 of its row);
    // in memory that chunk, operand u = (L % 4) / 2 of half h = L % 2 of the wave that wrote it, lies at
    // 1024 u + 16 (query + 32 h)
    lds_load_b128_once(store_descriptor(), x_lds + buf_load * kStoredTileBytes + it * 1024,
                       (uint32_t)(1024 * ((lane >> 1) & 1) + 16 * (16 * it + (lane >> 2) + 32 * (lane & 1))));
    if (it == 1) {
      store_at += (uint64_t)(store_tile + 1) * kStoredPairBytes;
      ++store_tile;
      buf_load = next_buffer(buf_load);
    }
  };

  // transposed operands of the tiles of Q and dO (the passes above read them the same way)
  typedef short Short4 __attribute__((ext_vector_type(4)));
  // Transposed operand (u, ib): 16 queries u of block feature_half * kHalfBlocks + ib of 32 features; two reads
  // (jj) each. tr_lane[ib][jj]: the lane's byte offset in the tile, the row of the read apart.
  uint32_t tr_lane[kHalfBlocks][2], x_lane;
  {
    const int j = lane & 15, group = lane >> 4;
    const int kq = j >> 2, fb = j & 3, hh = group >> 1, fg = group & 1;
#pragma unroll
    for (int ib = 0; ib < kHalfBlocks; ++ib) {
      const int i = feature_half * kHalfBlocks + ib;
      if constexpr (kQuads) {
        // row 16 u + 8 jj + 4 hh + kq, chunk 4 i + w of it, w = 2 fg + fb / 2: f is 4 kq + 2 jj + hh, so the chunk
        // lies at 16 (i / 4) + 4 (i % 4 ^ kq) + (w ^ hh ^ 2 jj)
        const uint32_t own = (uint32_t)(4 * hh + kq) * kRowBytes + 64u * (uint32_t)kq +
                             16u * (uint32_t)((2 * fg + (fb >> 1)) ^ hh) + 8u * (uint32_t)(fb & 1);
#pragma unroll
        for (int jj = 0; jj < 2; ++jj)
          tr_lane[ib][jj] = (own ^ (uint32_t)(64 * (i & 3) + 32 * jj)) + 256u * (uint32_t)(i >> 2);
      } else {
        const int flow = ((kq << 1) | hh) & kSwizzle;
        const int x = (2 * fg + (fb >> 1)) ^ (flow & 3);
        const int flip = flow >> 2;
        const uint32_t base = (uint32_t)(4 * hh + kq) * kRowBytes + (uint32_t)x * 16u + (uint32_t)(fb & 1) * 8u;
        tr_lane[ib][0] = tr_lane[ib][1] = base + 64u * (uint32_t)(flip ^ (i & 1)) + 64u * (uint32_t)(i & ~1);
      }
    }
    // the same read of a stored tile: rows of 64 bytes, no permutation of chunks
    x_lane = (uint32_t)(4 * hh + kq) * 64u + (uint32_t)fg * 32u + (uint32_t)fb * 8u;
  }
  auto read_transposed = [&](const T *base, int n) __attribute__((always_inline)) {
    const int u = n / kHalfBlocks, ib = n % kHalfBlocks;
    Short4 part[2];
#pragma unroll
    for (int jj = 0; jj < 2; ++jj) {
      const char *at = reinterpret_cast<const char *>(base) + tr_lane[ib][jj] + (16 * u + 8 * jj) * kRowBytes;
      part[jj] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) Short4 *)(at));
    }
    return __builtin_bit_cast(Frag, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
  };
  auto read_stored = [&](const unsigned char *base, int u) __attribute__((always_inline)) {
    Short4 part[2];
#pragma unroll
    for (int jj = 0; jj < 2; ++jj)
      part[jj] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) Short4 *)(base + x_lane + (16 * u + 8 * jj) * 64));
    return __builtin_bit_cast(Frag, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
  };

  f32x16 acc[2][kHalfBlocks]; // [key tile of the pair][block of features]
#pragma unroll
  for (int g = 0; g < 2; ++g)
#pragma unroll
    for (int i = 0; i < kHalfBlocks; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[g][i][r] = 0.f;

  constexpr int kRing = kOperands < 4 ? kOperands : 4;
  constexpr int kPerOperand = (kItems + kOperands - 1) / kOperands;
  // A tile as one straight run of code: operands are read from LDS kRing
  // operands ahead, a later tile's loads go between the products.
  auto one_tile = [&]() __attribute__((always_inline)) {
    const T *bt = t_lds + buf_now * kTile;
    const unsigned char *bx = x_pair + buf_now * kStoredTileBytes;
    Frag x[2][2], ring[kRing];
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int u = 0; u < 2; ++u) x[g][u] = read_stored(bx + g * (kStoredBuffers * kStoredTileBytes), u);
#pragma unroll
    for (int p = 0; p < kRing; ++p) ring[p] = read_transposed(bt, p);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < kOperands; ++n) {
      const int u = n / kHalfBlocks, ib = n % kHalfBlocks;
      acc[0][ib] = Op::run(ring[n % kRing], x[0][u], acc[0][ib]);
      acc[1][ib] = Op::run(ring[n % kRing], x[1][u], acc[1][ib]);
      if (n + kRing < kOperands) ring[n % kRing] = read_transposed(bt, n + kRing);
#pragma unroll
      for (int it = n * kPerOperand; it < (n + 1) * kPerOperand && it < kItems; ++it) stage_item(it);
      __builtin_amdgcn_sched_barrier(0);
    }
    buf_now = next_buffer(buf_now);
  };
  // the first tiles on their way
#pragma unroll
  for (int rep = 0; rep < kStoredBuffers - 1; ++rep)
#pragma unroll
    for (int it = 0; it < kItems; ++it) stage_item(it);
  // (Two tiles between barriers, with four buffers, measured slower: 413-445 against 352-391 us.)
  for (; t < tiles; ++t) {
    wait_vm<(kStoredBuffers - 2) * kItems>(); // (the tiles after t may still be on their way)
    __syncthreads(); // tile t is in LDS; the buffers written next (tile t - 1's) have been read
    one_tile();
  }
  wait_vm<0>(); // (nothing may still be on its way into LDS when the block ends)

  typedef T Out4 __attribute__((ext_vector_type(4)));
  const Strides3 &st_out = for_dv ? a.sdv : a.sdk;
  const float factor = for_dv ? (a.drop.drop ? a.drop.keep_scale : 1.0f) : a.scale;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    // lane c holds the key at slot c of the store's rows: c with bits 2 and 3 swapped
    const int own = own0 + 32 * ((wave & ~1) + g) + ((col & 0x13) | ((col & 4) << 1) | ((col & 8) >> 1));
    if (own >= S) continue;
    T *op = static_cast<T *>(for_dv ? a.dv : a.dk) + b * st_out.b + hd * st_out.h + (int64_t)own * st_out.s +
            32 * kHalfBlocks * feature_half;
#pragma unroll
    for (int i = 0; i < kHalfBlocks; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        Out4 w;
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) w[tt] = static_cast<T>(acc[g][i][4 * j + tt] * factor);
        *reinterpret_cast<Out4 *>(op + 32 * i + 8 * j + 4 * half) = w;
      }
  }
}


// dK and dV of the heads [a.bh0, a.bh0 + 8 * a.head_groups) from the tile store
template <typename T, int D>
int launch_stored(const BwdArgs &a, hipStream_t stream) {
  const int key_blocks = (a.S + 32 * stored_waves(D) - 1) / (32 * stored_waves(D));
  const dim3 grid((unsigned)(2 * 8 * a.head_groups * key_blocks)); // a block per gradient
  constexpr unsigned kLds = stored_lds_bytes<T, D>();
  auto *kernel = a.window > 0 ? attention_bwd_stored_kernel<T, D, true> : attention_bwd_stored_kernel<T, D, false>;
  if (kLds > 64u * 1024u) {
    const int s = raise_lds_limit(reinterpret_cast<const void *>(kernel), kLds, "oslo_attention_prefill_bwd_stored");
    if (s != OSLO_OK) return s;
  }
  kernel<<<grid, dim3(stored_waves(D) * kWave), kLds, stream>>>(a);
  return check_launch("attention_prefill_bwd_stored");
}

template <typename T, int D>
int launch_bwd_dim(const BwdArgs &a, float *delta, const void *out, const Strides3 &so,
                   hipStream_t stream, size_t store_bytes) {
  const int64_t rows = (int64_t)a.batch_heads * a.S;
  constexpr int kRows = kBlockThreads / (D / 8);
  attention_delta_kernel<T, D><<<dim3((unsigned)((rows + kRows - 1) / kRows)), dim3(kBlockThreads), 0, stream>>>(
      delta, static_cast<const T *>(out), static_cast<const T *>(a.dout), so, a.sdo, a.S, a.heads, rows);
  int s = check_launch("attention_prefill_bwd(delta)");
  if (s != OSLO_OK) return s;
  if (a.tiles != nullptr) {
    // The probabilities through memory: the dQ pass writes P and dS of every tile
    // on or below the diagonal, a second pass accumulates dK and dV from them (5
    // matrix products per tile, the number the mathematics has). Groups of 8
    // heads, as many at a time as the store holds, in launches of equal size.
    const int64_t per_group = 8 * a.head_tiles * kStoredPairBytes;
    const int fit = (int)std::min<int64_t>((int64_t)(store_bytes / (size_t)per_group), a.head_groups);
    const int launches = (a.head_groups + fit - 1) / fit;
    const int each = (a.head_groups + launches - 1) / launches;
    for (int g = 0; g < a.head_groups; g += each) {
      BwdArgs part = a;
      part.bh0 = 8 * g;
      part.head_groups = std::min(each, a.head_groups - g);
      s = launch_role<T, D, kRoleDQ, true>(part, stream);
      if (s != OSLO_OK) return s;
      s = launch_stored<T, D>(part, stream);
      if (s != OSLO_OK) return s;
    }
    return OSLO_OK;
  }
  s = launch_role<T, D, kRoleDQ>(a, stream);
  if (s != OSLO_OK) return s;
  // dK and dV: one combined pass where both accumulators fit a lane's registers
  // (heads of 64 and 128 features: 2 x 32 and 2 x 64 accumulator registers; timed
  // at [8,32,2048,64] 692 against 816 us for the whole backward, at [8,16,2048,128]
  // 635 against 648, with dropout 778 against 873). At 256 features they are 2 x
  // 128 beside 128 registers of fixed operands: the compiler spills 47 to 178
  // registers per lane, 39 scratch accesses in every tile, and the backward takes
  // 2917 us instead of 1382; there each gradient keeps a pass of its own.
  if constexpr (D <= OSLO_BWD_COMBINED_MAX_DIM) {
    return launch_role<T, D, kRoleDKV>(a, stream);
  } else {
    s = launch_role<T, D, kRoleDK>(a, stream);
    if (s != OSLO_OK) return s;
    return launch_role<T, D, kRoleDV>(a, stream);
  }
}

template <typename T>
int launch_bwd(const BwdArgs &a, float *delta, const void *out, const Strides3 &so, int head_dim,
               hipStream_t stream, size_t store_bytes) {
  switch (head_dim) {
    case 64: return launch_bwd_dim<T, 64>(a, delta, out, so, stream, store_bytes);
    case 128: return launch_bwd_dim<T, 128>(a, delta, out, so, stream, store_bytes);
    default: return launch_bwd_dim<T, 256>(a, delta, out, so, stream, store_bytes);
  }
}


} // namespace
} // namespace oslo

extern "C" size_t oslo_attention_prefill_bwd_workspace_bytes(int64_t batch, int64_t heads, int64_t S) {
  if (batch <= 0 || heads <= 0 || S <= 0) return 0;
  return (size_t)batch * (size_t)heads * (size_t)S * sizeof(float);
}

namespace oslo {

// Both entry points: `store` null = every pass computes the scores it needs.
static int prefill_bwd(const char *name, void *dq, void *dk, void *dv, const void *dout, const void *q, const void *k,
                const void *v, const void *out, const float *lse, float *workspace, void *store,
                size_t store_bytes, const float *pad, float scale, float p, uint64_t philox_seed,
                uint64_t philox_offset, int64_t batch, int64_t heads, int64_t S, int64_t head_dim,
                int64_t window, const int64_t *strides, int dtype, oslo_stream_t stream) {
  if (batch < 0 || heads < 0 || S < 0 || head_dim < 0 || window < 0)
    return fail(OSLO_E_BAD_ARG, "%s: negative size", name);
  if (dtype != OSLO_F16 && dtype != OSLO_BF16) {
    if (dtype == OSLO_F32) return fail(OSLO_E_UNSUPPORTED, "%s: fp16 and bf16 are taken, not fp32", name);
    return fail(OSLO_E_BAD_ARG, "unknown dtype %d", dtype);
  }
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(OSLO_E_UNSUPPORTED, "%s: heads of %lld features (64, 128 or 256 are taken)", name,
                (long long)head_dim);
  if (!(scale > 0.0f)) return fail(OSLO_E_BAD_ARG, "%s: the scale must be positive", name);
  DropArgs drop;
  const int ds = make_drop_args(name, p, philox_seed, philox_offset, &drop);
  if (ds != OSLO_OK) return ds;
  if (batch == 0 || heads == 0 || S == 0) return OSLO_OK;
  if (drop.drop && S % 8 != 0)
    return fail(OSLO_E_UNSUPPORTED, "%s: with attention dropout S must be a multiple of 8", name);
  if (!dq || !dk || !dv || !dout || !q || !k || !v || !out || !lse || !workspace || !strides)
    return fail(OSLO_E_BAD_ARG, "%s: null pointer", name);
  if (batch * heads > (int64_t)0x7fffffff / 8 || batch * heads * S > (int64_t)0x7fffffff)
    return fail(OSLO_E_UNSUPPORTED, "%s: too many rows for one launch", name);
  // strides: q, k, v, out, dout, dq, dk, dv (batch, head, position each)
  const void *ptrs[8] = {q, k, v, out, dout, dq, dk, dv};
  for (int i = 0; i < 8; ++i) {
    if (!aligned16(ptrs[i])) return fail(OSLO_E_UNSUPPORTED, "%s: tensors must be 16-byte aligned", name);
    const int64_t sb = strides[3 * i], sh = strides[3 * i + 1], ss = strides[3 * i + 2];
    if (sb < 0 || sh < 0 || ss < head_dim || sb % 8 || sh % 8 || ss % 8)
      return fail(OSLO_E_UNSUPPORTED,
                  "%s: strides must be multiples of 8 elements, the position stride at least head_dim", name);
    if ((S + kOwnPerBlock) * ss * 2 > (int64_t)0x7fffffff)
      return fail(OSLO_E_UNSUPPORTED, "%s: a head's slice exceeds 2 GiB", name);
  }
  if (pad != nullptr && (S % 4 != 0 || !aligned16(pad)))
    return fail(OSLO_E_UNSUPPORTED,
                "%s: with a padding mask S must be a multiple of 4 and the mask 16-byte aligned", name);
  if (!aligned16(lse) || !aligned16(workspace) || !aligned16(store))
    return fail(OSLO_E_UNSUPPORTED, "%s: lse and the workspaces must be 16-byte aligned", name);
  auto st = [&](int i) { return Strides3{strides[3 * i], strides[3 * i + 1], strides[3 * i + 2]}; };
  BwdArgs a;
  a.q = q, a.k = k, a.v = v, a.dout = dout, a.dq = dq, a.dk = dk, a.dv = dv;
  a.lse = lse, a.delta = workspace, a.pad = pad, a.drop = drop;
  a.sq = st(0), a.sk = st(1), a.sv = st(2), a.sdo = st(4), a.sdq = st(5), a.sdk = st(6), a.sdv = st(7);
  a.scale = scale;
  a.scale_log2e = scale * kLog2eB;
  a.S = (int)S;
  a.heads = (int)heads;
  a.batch_heads = (int)(batch * heads);
  a.head_groups = (a.batch_heads + 7) / 8;
  a.own_blocks = (int)((S + kOwnPerBlock - 1) / kOwnPerBlock);
  a.window = window >= S ? 0 : (int)window;
  a.tiles = static_cast<unsigned char *>(store);
  a.bh0 = 0;
  a.head_tiles = stored_head_tiles(a.own_blocks);

  if (store != nullptr && store_bytes < (size_t)(8 * a.head_tiles * kStoredPairBytes))
    return fail(OSLO_E_BAD_ARG, "%s: a store of %zu bytes; 8 heads of %lld positions need %lld", name, store_bytes,
                (long long)S, (long long)(8 * a.head_tiles * kStoredPairBytes));
  if ((int64_t)16 * a.head_groups * a.own_blocks > (int64_t)0x7fffffff)
    return fail(OSLO_E_UNSUPPORTED, "%s: too many blocks for one launch", name);
  hipStream_t stm = static_cast<hipStream_t>(stream);
  if (dtype == OSLO_F16) return launch_bwd<f16>(a, workspace, out, st(3), (int)head_dim, stm, store_bytes);
  return launch_bwd<bf16>(a, workspace, out, st(3), (int)head_dim, stm, store_bytes);
}

} // namespace oslo

extern "C" size_t oslo_attention_prefill_bwd_store_bytes(int64_t batch, int64_t heads, int64_t S) {
  if (batch <= 0 || heads <= 0 || S <= 0) return 0;
  const int64_t groups = (batch * heads + 7) / 8;
  const int64_t own_blocks = (S + oslo::kOwnPerBlock - 1) / oslo::kOwnPerBlock;
  return (size_t)(8 * groups) * (size_t)oslo::stored_head_tiles(own_blocks) * (size_t)oslo::kStoredPairBytes;
}

extern "C" int oslo_attention_prefill_bwd(void *dq, void *dk, void *dv, const void *dout,
                                          const void *q, const void *k, const void *v,
                                          const void *out, const float *lse,
                                          float *workspace, const float *pad, float scale,
                                          float p, uint64_t philox_seed,
                                          uint64_t philox_offset,
                                          int64_t batch, int64_t heads, int64_t S,
                                          int64_t head_dim, int64_t window,
                                          const int64_t *strides, int dtype,
                                          oslo_stream_t stream) {
  return oslo::prefill_bwd("oslo_attention_prefill_bwd", dq, dk, dv, dout, q, k, v, out, lse, workspace, nullptr, 0,
                           pad, scale, p, philox_seed, philox_offset, batch, heads, S, head_dim, window, strides,
                           dtype, stream);
}

extern "C" int oslo_attention_prefill_bwd_stored(void *dq, void *dk, void *dv, const void *dout,
                                                 const void *q, const void *k, const void *v,
                                                 const void *out, const float *lse,
                                                 float *workspace, void *store, size_t store_bytes,
                                                 const float *pad, float scale,
                                                 float p, uint64_t philox_seed,
                                                 uint64_t philox_offset,
                                                 int64_t batch, int64_t heads, int64_t S,
                                                 int64_t head_dim, int64_t window,
                                                 const int64_t *strides, int dtype,
                                                 oslo_stream_t stream) {
  if (store == nullptr)
    return oslo::fail(OSLO_E_BAD_ARG, "oslo_attention_prefill_bwd_stored: null store");
  return oslo::prefill_bwd("oslo_attention_prefill_bwd_stored", dq, dk, dv, dout, q, k, v, out, lse, workspace, store,
                           store_bytes, pad, scale, p, philox_seed, philox_offset, batch, heads, S, head_dim, window,
                           strides, dtype, stream);
}

