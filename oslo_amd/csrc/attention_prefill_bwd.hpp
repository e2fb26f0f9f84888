// Backward of the one-kernel causal prompt attention (attention_prefill.hip):
// dQ, dK and dV from Q, K, V, dO, the forward's output O and the log-sum-exp
// of every row, without the [S, S] matrices in memory (or, for the entry
// point with a tile store, with their tiles below the diagonal in a workspace
// between two passes of one call). With
//   P  = exp2(scale*log2e * Q K^T + pad*log2e - lse)      (the probabilities)
//   dP = dO V^T,   delta[q] = sum_d dO[q,d] * O[q,d]
//   dS = scale * P o (dP - delta)
// the gradients are dV = P^T dO, dQ = dS K, dK = dS^T Q. It replaces, for
// training, the backward of the three launches of the reference's fused
// attention (oslo/models/gptj/modeling_gptj.py:936-951: matmul, softmax
// kernel, matmul, differentiated by autograd), which keeps the probabilities
// and their gradient as [B, H, S, S] tensors.
//
// One kernel template serves every gradient. A block owns 128 positions (32
// per wave, one per lane of each half) and walks over the positions of the
// other kind in tiles: for dQ it owns queries and walks the keys up to the
// diagonal, for dK and dV it owns keys and walks the queries from the
// diagonal on. Both score-like products put the own position in the lane:
//   T1[other, own] = Other1 (A operand, LDS, rows = other) x Own1^T (B, fixed)
//   T2[other, own] = Other2 (A operand, LDS)               x Own2^T (B, fixed)
// (dQ: T1 = K Q^T = S^T, T2 = V dO^T = dP^T; dK/dV: T1 = Q K^T = S, T2 = dO V^T
// = dP), so P and dS come out in the accumulator layout of
// v_mfma_f32_32x32x16, which is also the B-operand layout of the accumulating
// products
//   Acc^T[d, own] += OtherT (A operand, LDS, rows = features) x X[other, own]
// (dQ^T += K^T dS^T; dK^T += Q^T dS; dV^T += dO^T P) once the contraction
// order is permuted the way the forward does it for V^T. Quantities indexed by
// the own position are per-lane scalars, those indexed by the other position
// are read per tile from LDS. Each block sums in a fixed order and no two
// blocks write the same element: the gradients are deterministic. The price is
// that scores are computed once per owner kind: dQ takes three matrix products
// per visible (query, key) tile and dK and dV together four (7 instead of 5)
// where one pass can hold both accumulators (heads of 64 and 128 features);
// at 256 features dK takes three and dV two in passes of their own (8).
//
// The kernel is built the way the forward is: tiles of 32 positions of the
// other kind loaded straight into LDS (four buffers per tensor), stored as they
// are in memory, read as A operands of the score-like products 16 bytes per
// lane and as A operands of the accumulating product through the transposing
// read (no transposed copy, no staging through registers); a tile's code is
// ordered by hand: the products of T1, those of T2, then the accumulating
// products of the previous tile with this tile's probabilities and score
// gradients worked out between them. One permutation of a row's 16-byte chunks
// serves both reads (f(row) below).

#pragma once

#include "attention.hpp"

namespace oslo {
namespace {

// Largest head size whose dK and dV share a pass (a build switch for
// measurements: 256 compiles the combined pass there too, where it spills).
#ifndef OSLO_BWD_COMBINED_MAX_DIM
#define OSLO_BWD_COMBINED_MAX_DIM 128
#endif
// Waves of a block of the pass that reads the tile store (32 keys each), heads
// of 128 and 256 features (a build switch for measurements: 4 or 8).
#ifndef OSLO_STORED_WAVES
#define OSLO_STORED_WAVES 8
#endif

constexpr int kOwnPerBlock = 128;
constexpr float kLog2eB = 1.4426950408889634f;

// kRoleDKV: dK and dV in one pass (both own keys and walk queries: the scores
// and the probabilities are computed once for the two, 4 products per tile
// where the two passes have 5; it needs both accumulators in registers).
enum Role { kRoleDQ = 0, kRoleDK = 1, kRoleDV = 2, kRoleDKV = 3 };

// Blocks per CU the kernel is compiled for (a wave per SIMD each).
constexpr int bwd_blocks_per_cu(int D, int role) {
  if (role == kRoleDKV) return D == 256 ? 1 : D == 128 ? 1 : 2;
  return D == 256 ? 1 : D == 128 ? 2 : 3;
}

struct Strides3 {
  int64_t b, h, s; // element strides: batch, head, position
};

struct BwdArgs {
  const void *q, *k, *v, *dout;
  void *dq, *dk, *dv;
  const float *lse;   // [batch * heads, S], log2 units, from the forward
  const float *delta; // [batch * heads, S]
  const float *pad;   // [batch, S] additive, or null
  Strides3 sq, sk, sv, sdo, sdq, sdk, sdv;
  float scale, scale_log2e;
  int S, heads, batch_heads, head_groups, own_blocks, window;
  DropArgs drop; // attention dropout of the forward (the DROP variants)
  // The passes that exchange the probabilities through memory (below): the
  // tile store, the first head of the launch (a launch covers the heads
  // [bh0, bh0 + 8 * head_groups) below batch_heads; tiles of head bh0 come
  // first in the store), and the number of tiles a head has there.
  unsigned char *tiles;
  int bh0;
  int64_t head_tiles;
  // The PACKED variant: the sequences; the forward's output, from which the pass that owns queries works
  // out delta itself (and leaves it for the passes that own keys); and the entries whose group of
  // query heads is shared by `parts` blocks (the first `split` of the list: those with most queries),
  // which leave fp32 sums [entry * parts + part][kv head][dK, dV][128][D] in `partial`.
  PackedArgs packed;
  const void *out, *out_low; // (out_low: null, or what rounding left out of it)
  Strides3 sout;
  float *delta_out;
  float *partial;
  int split, parts;
};

// The tile store. P (after dropout) and dS / scale of the 32 queries x 32 keys of
// query tile Qb and key tile Kb <= Qb of a head are 2 KiB each, one behind the
// other at tile index Qb (Qb + 1) / 2 + Kb, each as the pass that computes
// them holds it: [operand u][lane][8 values], the B operand u = 0, 1 of that
// pass's own accumulating product of lane (query, half h), whose value i is
// key 16 u + 8 (i / 4) + 4 h + i % 4: a store instruction of a wave writes 1 KiB
// in a row. The pass that consumes them gathers a tile into LDS as rows of
// [query][slot], slot 16 u + 8 h + i, and reads it through the transposing LDS
// read, key slot in the lane.
constexpr int kStoredTileBytes = 2048;                      // one of the two
constexpr int kStoredPairBytes = 2 * kStoredTileBytes;      // P, then dS
__host__ __device__ constexpr int64_t stored_head_tiles(int64_t own_blocks) {
  const int64_t n = own_blocks * (kOwnPerBlock / 32);
  return n * (n + 1) / 2;
}

constexpr int kSchedTile = 32;
constexpr int kSchedBuffers = 4;

template <typename T, int D, int ROLE>
constexpr unsigned sched_lds_bytes() {
  return 2u * kSchedBuffers * kSchedTile * D * sizeof(T) + kSchedBuffers * 2u * 256u * sizeof(float) +
         kWavesPerBlock * 32u * sizeof(uint32_t);
}

template <typename T, int D, int ROLE, bool HAS_PAD, bool HAS_WINDOW, bool DROP, bool STORE = false, bool PACKED = false>
__global__ __launch_bounds__(kBlockThreads, bwd_blocks_per_cu(D, ROLE)) void attention_bwd_kernel(
    const BwdArgs a) {
  static_assert(ROLE >= kRoleDQ && ROLE <= kRoleDKV, "unknown pass");
  static_assert(!STORE || ROLE == kRoleDQ, "the pass that owns queries writes the tile store");
  static_assert(!PACKED || (!HAS_PAD && !DROP && !STORE), "packed sequences: no padding mask, no dropout, no tile store");
  using Op = MatrixOp<T>;
  using Frag = typename Op::Frag;
  constexpr bool kKeysOwn = ROLE != kRoleDQ;
  constexpr bool kNeedT2 = ROLE != kRoleDV;
  constexpr bool kTwoAcc = ROLE == kRoleDKV; // acc = dK^T, acc2 = dV^T
  constexpr bool kKeepP = kTwoAcc || STORE;  // the probabilities are wanted beside dS
  constexpr int kChunks = D / 8;   // 16-byte chunks of a position
  constexpr int kSteps = D / 16;   // contraction steps over the features
  constexpr int kBlocksD = D / 32; // 32-row blocks of the accumulator
  constexpr int kLoadsN = kSchedTile * kChunks / kBlockThreads; // loads per thread and tile of a tensor
  constexpr int kTile = kSchedTile * D; // elements
  constexpr int kRowBytes = D * (int)sizeof(T);
  constexpr int kSwizzle = kChunks >= 16 ? 15 : 7;
  constexpr int kRowSlots = 256; // floats of a tile's per-position values: the first 32 count

  extern __shared__ __align__(1024) unsigned char lds_raw[];
  T *const o1_lds = reinterpret_cast<T *>(lds_raw);            // [4][position][chunk ^ f(position)][8]
  T *const o2_lds = o1_lds + kSchedBuffers * kTile;            // the same for the second tensor
  // per-position values of a tile: queries: log-sum-exp and delta; keys: the padding mask's value
  float *const rows_lds = reinterpret_cast<float *>(o2_lds + kSchedBuffers * kTile); // [4][2][256]

  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int half = lane >> 5;
  const int col = lane & 31;
  uint32_t *const keep_lds =
      reinterpret_cast<uint32_t *>(rows_lds + kSchedBuffers * 2 * kRowSlots) + 32 * wave; // a wave's keep bits of a tile

  // PACKED: the sequence comes from the list of blocks. A block that owns
  // queries takes one query head; one that owns keys takes a key/value head and
  // walks the queries of every head of its group in turn, so that the sums over the
  // group stay in registers.
  int bh, b, hd, kv_hd, S, own_block;
  int64_t start = 0;   // the sequence's first token
  int64_t packed_row = 0; // the (first) query head's row of per-position values
  int64_t stat_step = 0; // from a query head's row to the next head's
  int group_heads = 1;   // query heads the block walks
  int64_t part_slot = -1; // of its fp32 sums, if it walks a part of the group only
  if constexpr (PACKED) {
    const unsigned per_entry = kKeysOwn ? (unsigned)a.packed.kv_heads : (unsigned)a.heads;
    const int r = (int)(blockIdx.x % per_entry);
    unsigned entry = blockIdx.x / per_entry;
    int first_head = 0; // of the group
    if constexpr (kKeysOwn) {
      group_heads = a.packed.group;
      const unsigned shared = (unsigned)(a.split * a.parts);
      if (entry < shared) {
        const int part = (int)(entry % (unsigned)a.parts);
        part_slot = (int64_t)entry * a.packed.kv_heads + r;
        first_head = part * a.packed.group / a.parts;
        group_heads = (part + 1) * a.packed.group / a.parts - first_head;
        entry /= (unsigned)a.parts;
      } else {
        entry -= shared - (unsigned)a.split;
      }
    }
    const PackedBlock e = packed_block(a.packed, entry);
    if (!packed_block_in_range(a.packed, e, kOwnPerBlock)) return; // the whole block
    b = 0;
    hd = kKeysOwn ? r * a.packed.group + first_head : packed_query_head(a.packed, r);
    kv_hd = kKeysOwn ? r : hd / a.packed.group;
    bh = hd;
    S = e.length;
    own_block = e.block;
    start = e.start;
    packed_row = hd * a.packed.tokens + start;
    stat_step = a.packed.tokens;
  } else {
    const int xcd = blockIdx.x & 7;
    const int slot = blockIdx.x >> 3;
    bh = a.bh0 + xcd + 8 * (slot % a.head_groups);
    const int idx = slot / a.head_groups;
    own_block = kKeysOwn ? idx : a.own_blocks - 1 - idx;
    if (bh >= a.batch_heads) return; // the whole block
    b = bh / a.heads;
    hd = kv_hd = bh - b * a.heads;
    S = a.S;
  }
  const int own0 = own_block * kOwnPerBlock;
  const int wave_own0 = own0 + 32 * wave;
  const int own = wave_own0 + col;

  auto slice = [&](const void *p, const Strides3 &st, int head) __attribute__((always_inline)) {
    return static_cast<const T *>(p) + b * st.b + head * st.h + start * st.s;
  };
  auto slice_bytes = [&](const Strides3 &st) __attribute__((always_inline)) {
    return (uint32_t)(((int64_t)(S - 1) * st.s + D) * sizeof(T));
  };
  const Strides3 &st_own1 = kKeysOwn ? a.sk : a.sq;
  const Strides3 &st_own2 = kKeysOwn ? a.sv : a.sdo;
  const Strides3 &st_o1 = kKeysOwn ? a.sq : a.sk;
  const Strides3 &st_o2 = kKeysOwn ? a.sdo : a.sv;
  const T *own1_p = slice(kKeysOwn ? a.k : a.q, st_own1, kKeysOwn ? kv_hd : hd);
  const T *own2_p = slice(kKeysOwn ? a.v : a.dout, st_own2, kKeysOwn ? kv_hd : hd);
  const T *o1_p = slice(kKeysOwn ? a.q : a.k, st_o1, kKeysOwn ? hd : kv_hd);
  const T *o2_p = slice(kKeysOwn ? a.dout : a.v, st_o2, kKeysOwn ? hd : kv_hd);
  const uint32_t o1_row = (uint32_t)st_o1.s * sizeof(T);
  const uint32_t o2_row = (uint32_t)st_o2.s * sizeof(T);

  // B operands of the own positions, in registers for the whole kernel
  Frag own1[kSteps], own2[kNeedT2 ? kSteps : 1];
  {
    const BufRsrc rs1 = make_rsrc(own1_p, slice_bytes(st_own1));
    const uint32_t row1 = (uint32_t)st_own1.s * sizeof(T);
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      own1[s] = __builtin_bit_cast(Frag, __builtin_amdgcn_raw_buffer_load_b128(
                                             rs1, (uint32_t)own * row1 + (uint32_t)(16 * s + 8 * half) * sizeof(T), 0, 0));
    if constexpr (kNeedT2) {
      const BufRsrc rs2 = make_rsrc(own2_p, slice_bytes(st_own2));
      const uint32_t row2 = (uint32_t)st_own2.s * sizeof(T);
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        own2[s] = __builtin_bit_cast(Frag, __builtin_amdgcn_raw_buffer_load_b128(
                                               rs2, (uint32_t)own * row2 + (uint32_t)(16 * s + 8 * half) * sizeof(T), 0, 0));
    }
  }
  const int64_t stat_row = PACKED ? packed_row : (int64_t)bh * S;
  float own_lse = 0.f, own_delta = 0.f, own_pad = 0.f; // (the padding value, floored)
  // PACKED, own queries: the rows of O, from which delta is worked out while the first
  // tiles are on their way (the loads are issued here)
  constexpr bool kOwnDelta = PACKED && !kKeysOwn;
  Frag own_o[kOwnDelta ? kSteps : 1], own_low[kOwnDelta ? kSteps : 1];
  if constexpr (kOwnDelta) {
    const BufRsrc rs = make_rsrc(slice(a.out, a.sout, hd), slice_bytes(a.sout));
    const uint32_t row = (uint32_t)a.sout.s * sizeof(T);
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      own_o[s] = __builtin_bit_cast(Frag, __builtin_amdgcn_raw_buffer_load_b128(
                                              rs, (uint32_t)own * row + (uint32_t)(16 * s + 8 * half) * sizeof(T), 0, 0));
    const BufRsrc low = make_rsrc(slice(a.out_low, a.sout, hd), a.out_low != nullptr ? slice_bytes(a.sout) : 0u); // (null: zeros)
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      own_low[s] = __builtin_bit_cast(Frag, __builtin_amdgcn_raw_buffer_load_b128(
                                                low, (uint32_t)own * row + (uint32_t)(16 * s + 8 * half) * sizeof(T), 0, 0));
    if (own < S) own_lse = a.lse[stat_row + own];
  } else if constexpr (!kKeysOwn) {
    if (own < S) {
      own_lse = a.lse[stat_row + own];
      own_delta = a.delta[stat_row + own];
    }
  } else if constexpr (HAS_PAD) {
    if (own < S) own_pad = fmaxf(a.pad[(int64_t)b * S + own], kMaskFloor);
  }

  // Tiles [first_tile, tiles) of the other kind this block walks. Those before
  // masked_until and those from plain_until on may hold pairs that are not
  // visible; the tiles between them are visible in full to every own position.
  // Own queries: the causal boundary crosses the last four tiles, the edges of
  // the queries' windows the first ones. Own keys: the boundary crosses the
  // first four; a window ends the walk at the last query that sees the block's
  // last key, and its edge crosses the tiles from the first query that no
  // longer sees the block's first key on.
  const int window = HAS_WINDOW ? a.window : 0;
  int first_tile, tiles, masked_until, plain_until;
  if constexpr (!kKeysOwn) {
    const int last_key = (own0 + kOwnPerBlock < S ? own0 + kOwnPerBlock : S) - 1;
    tiles = last_key / kSchedTile + 1;
    first_tile = HAS_WINDOW && own0 - window + 1 > 0 ? (own0 - window + 1) / kSchedTile : 0;
    masked_until = HAS_WINDOW && own0 + kOwnPerBlock - window > 0
                       ? (own0 + kOwnPerBlock - window + kSchedTile - 1) / kSchedTile
                       : 0;
    plain_until = own0 / kSchedTile;
  } else {
    first_tile = own0 / kSchedTile;
    int last_query = S - 1;
    if (HAS_WINDOW && own0 + kOwnPerBlock - 1 + window - 1 < last_query) last_query = own0 + kOwnPerBlock - 1 + window - 1;
    tiles = last_query / kSchedTile + 1;
    masked_until = first_tile + kOwnPerBlock / kSchedTile;
    plain_until = HAS_WINDOW ? (own0 + window) / kSchedTile : tiles;
  }
  if (masked_until > tiles) masked_until = tiles;
  if (plain_until > tiles) plain_until = tiles;

  // The permutation of a row's chunks: chunk c of row r lies at c ^ f(r). The
  // 16 lanes that read 16 consecutive rows at one chunk (natural operands) must
  // get 16 values of f, the 16 lanes of a transposing read (rows 4c .. 4c + 3,
  // two chunks, both halves of each) four values that differ above bit 0: f
  // puts the row's two low bits at bits 1 and 2, bit 2 at bit 0, bit 3 stays.
  // (At 256 features, where the registers for eight lane offsets are there, f is
  // 4 (r % 4) + r / 4 % 4 instead: the four rows of a transposing read then use four
  // different quarters of the banks for both 16-feature halves at once; with the
  // f above two of the four share theirs, two more cycles for every such read.)
  constexpr bool kQuads = D == 256;
  auto f_of = [](int r) __attribute__((always_inline)) {
    if (kQuads) return ((r & 3) << 2) | ((r >> 2) & 3);
    return (((r & 3) << 1) | ((r >> 2) & 1) | (r & 8)) & kSwizzle;
  };
  uint32_t o1_off[kLoadsN], o2_off[kLoadsN];
#pragma unroll
  for (int j = 0; j < kLoadsN; ++j) {
    const int sigma = (4 * j + wave) * kWave + lane;
    const int row = sigma / kChunks, at = sigma % kChunks;
    o1_off[j] = (uint32_t)row * o1_row + (uint32_t)(at ^ f_of(row)) * 16u;
    o2_off[j] = (uint32_t)row * o2_row + (uint32_t)(at ^ f_of(row)) * 16u;
  }
  const uint32_t row_off = tid < kSchedTile ? (uint32_t)tid * 4u : 0x80000000u;
  TileStream o1_src, o2_src, lse_src, delta_src; // the next tile to load (tile t + 2 while tile t is computed)
  auto start_sources = [&](const T *first, const T *second, int64_t row) __attribute__((always_inline)) {
    o1_src.start(first, slice_bytes(st_o1), o1_row, kSchedTile, first_tile, tiles);
    o2_src.start(second, slice_bytes(st_o2), o2_row, kSchedTile, first_tile, tiles);
    if constexpr (kKeysOwn) {
      lse_src.start(a.lse + row, (uint32_t)S * 4u, 4u, kSchedTile, first_tile, tiles);
      if constexpr (kNeedT2) delta_src.start(a.delta + row, (uint32_t)S * 4u, 4u, kSchedTile, first_tile, tiles);
    } else if constexpr (HAS_PAD) { // the keys' mask values take the first of the two rows
      lse_src.start(a.pad + (int64_t)b * S, (uint32_t)S * 4u, 4u, kSchedTile, first_tile, tiles);
    }
  };
  constexpr int kRowItems = kKeysOwn ? (kNeedT2 ? 2 : 1) : HAS_PAD ? 1 : 0; // (the dV pass needs no delta)
  constexpr int kItems = 2 * kLoadsN + kRowItems;
  constexpr int kLoadsPerTile = kItems;
  int t = first_tile;
  // buffer of tile t + d
  auto buffer_of = [&](int d) __attribute__((always_inline)) { return (t + d) & (kSchedBuffers - 1); };
  // item `it` of the staging of tile t: the loads of tile t + 2
  auto stage_item = [&](int it) __attribute__((always_inline)) {
    const int buf = buffer_of(2);
    if (it < kLoadsN) {
      lds_load_b128(o1_src.descriptor(), o1_lds + buf * kTile + (4 * it + wave) * (kWave * 8), o1_off[it]);
      if (it == kLoadsN - 1) o1_src.advance();
      return;
    }
    it -= kLoadsN;
    if (it < kLoadsN) {
      lds_load_b128(o2_src.descriptor(), o2_lds + buf * kTile + (4 * it + wave) * (kWave * 8), o2_off[it]);
      if (it == kLoadsN - 1) o2_src.advance();
      return;
    }
    it -= kLoadsN;
    if constexpr (kRowItems > 0) {
      // every wave loads 64 values into a quarter of its own; the first 32 of the first wave's count
      float *dst = rows_lds + (buf * 2 + it) * kRowSlots + wave * kWave;
      if (it == 0) {
        lds_load_b32(lse_src.descriptor(), dst, row_off);
        lse_src.advance();
      } else {
        lds_load_b32(delta_src.descriptor(), dst, row_off);
        delta_src.advance();
      }
    }
  };

  // natural operand s of the tile in `base`: lane (row, half) takes chunk 2 s + half of its row
  const uint32_t nat_lane = (uint32_t)col * kRowBytes + (uint32_t)((half ^ f_of(col)) << 4);
  auto read_natural = [&](const T *base, int s) __attribute__((always_inline)) {
    return *reinterpret_cast<const Frag *>(reinterpret_cast<const char *>(base) + (nat_lane ^ (uint32_t)(s << 5)));
  };
  // Transposed operand n (16 positions u into block i of 32 features): of 16
  // lanes, lane j points at 8 bytes (4 features) of position j / 4; lane i gets
  // back feature i of the four positions. Two reads make an operand: slots 0..3
  // are positions 16u + 4h + 0..3, slots 4..7 positions 16u + 8 + 4h + 0..3 (h
  // the lane's half of the wave): the rows the accumulator layout gives a lane.
  typedef short Short4 __attribute__((ext_vector_type(4)));
  uint32_t tr_lane[kQuads ? 8 : 2]; // for even and odd blocks of 32 features (kQuads: per block % 4 and read of the two)
  {
    const int j = lane & 15, group = lane >> 4;
    const int kq = j >> 2, fb = j & 3, hh = group >> 1, fg = group & 1;
    if constexpr (kQuads) {
      // row 16 u + 8 jj + 4 hh + kq, chunk 4 i + w of it, w = 2 fg + fb / 2: f is 4 kq + 2 jj + hh, so the chunk lies
      // at 16 (i / 4) + 4 (i % 4 ^ kq) + (w ^ hh ^ 2 jj): the lane's part, with the read's i % 4 and jj folded in
      const uint32_t own_part = (uint32_t)(4 * hh + kq) * kRowBytes + 64u * (uint32_t)kq +
                                16u * (uint32_t)((2 * fg + (fb >> 1)) ^ hh) + 8u * (uint32_t)(fb & 1);
#pragma unroll
      for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int jj = 0; jj < 2; ++jj) tr_lane[2 * v + jj] = own_part ^ (uint32_t)(64 * v + 32 * jj);
    } else {
      // f of the lane's rows 16u + 8jj + 4hh + kq is 2 kq | hh | 8 jj; the part below bit 3:
      const int flow = ((kq << 1) | hh) & kSwizzle;
      const int x = (2 * fg + (fb >> 1)) ^ (flow & 3);
      const int flip = flow >> 2; // its bit 2 swaps neighbouring blocks of four chunks
      const uint32_t base = (uint32_t)(4 * hh + kq) * kRowBytes + (uint32_t)x * 16u + (uint32_t)(fb & 1) * 8u;
      tr_lane[0] = base + 64u * (uint32_t)flip;
      tr_lane[1] = base + 64u * (uint32_t)(1 ^ flip);
    }
  }
  auto read_transposed = [&](const T *base, int n) __attribute__((always_inline)) {
    const int u = n / kBlocksD, i = n % kBlocksD;
    Short4 part[2];
#pragma unroll
    for (int jj = 0; jj < 2; ++jj) {
      const char *at;
      if constexpr (kQuads) {
        at = reinterpret_cast<const char *>(base) + tr_lane[2 * (i & 3) + jj] + 256 * (i >> 2) + (16 * u + 8 * jj) * kRowBytes;
      } else {
        // rows with bit 3 set (jj = 1) have bit 3 of f set: blocks two apart swap (head sizes of 16 chunks and more)
        const int ii = kSwizzle >= 8 ? i ^ (2 * jj) : i;
        at = reinterpret_cast<const char *>(base) + tr_lane[ii & 1] + 64 * (ii & ~1) + (16 * u + 8 * jj) * kRowBytes;
      }
      part[jj] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) Short4 *)(at));
    }
    return __builtin_bit_cast(Frag, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
  };

  f32x16 acc[kBlocksD], acc2[kTwoAcc ? kBlocksD : 1];
#pragma unroll
  for (int i = 0; i < kBlocksD; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
  if constexpr (kTwoAcc) {
#pragma unroll
    for (int i = 0; i < kBlocksD; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc2[i][r] = 0.f;
  }
  // what the accumulating products take of the last tile computed: xf = P (dV
  // pass) or P o (dP - delta); in the combined pass xp = P as well
  Frag xf[2], xp[2];

  // which tensor the accumulating product reads transposed: K (dQ), Q (dK), dO (dV)
  auto transposed_tile = [&](int d) __attribute__((always_inline)) {
    return (ROLE == kRoleDV ? o2_lds : o1_lds) + buffer_of(d) * kTile;
  };
  auto transposed_tile2 = [&](int d) __attribute__((always_inline)) { return o2_lds + buffer_of(d) * kTile; }; // dO (combined pass)
  // slice `n` of `slices` of a tile's elementwise work: P = exp2(scale*log2e *
  // T1 + pad*log2e - lse), X = P (dV) or P (T2 - delta) (the scale goes onto
  // the result). With attention dropout the forward multiplied V with
  // keep * P / (1-p): the P product takes the kept probabilities (1/(1-p) goes
  // onto dV at the end), and the gradient of the dropped-out probabilities is
  // keep * dP / (1-p). The keep bits of the tile are drawn in the first slice.
  u32x4 keep_words[4];
  uint32_t keep_bits = 0;
  // The tile's per-position values of register r (row 8 (r / 4) + 4 half + r % 4
  // of the tile) are read kAhead registers before they are used: read where
  // they are used, every slice of the elementwise work would wait for the LDS.
  // (Not at head_dim 64, where the registers for it are not there.)
  constexpr bool kRowValues = kKeysOwn || HAS_PAD;
  constexpr int kAhead = D >= 128 ? 4 : 0;
  float row_a[16], row_b[16];
  auto read_row_values = [&](int r) __attribute__((always_inline)) {
    if constexpr (kRowValues) {
      const float *rows = rows_lds + buffer_of(0) * 2 * kRowSlots + 8 * (r >> 2) + 4 * half + (r & 3);
      row_a[r] = rows[0];
      if constexpr (kKeysOwn && kNeedT2) row_b[r] = rows[kRowSlots];
    }
  };
  auto elementwise = [&]<bool MASKED>(f32x16 &t1, f32x16 &t2, int n, int slices, Frag (&x)[2], Frag (&x2)[2])
                         __attribute__((always_inline)) {
    if constexpr (DROP) {
      if (n == 0) {
        const int other0 = t * kSchedTile;
        stage_keep_bits(keep_lds, a.drop, bh, S, kKeysOwn ? other0 : wave_own0, kKeysOwn ? wave_own0 : other0, lane);
        if constexpr (kKeysOwn) {
#pragma unroll
          for (int j = 0; j < 4; ++j) keep_words[j] = keep_words_key_lane(keep_lds, j, half);
        } else {
          keep_bits = keep_word_query_lane(keep_lds, col) >> (4 * half);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      if (r * slices / 16 != n) continue;
      const int rr = 8 * (r >> 2) + 4 * half + (r & 3); // the register's row of the tile
      if (r + kAhead < 16) read_row_values(r + kAhead);
      float shift, delta_r = own_delta;
      if constexpr (kKeysOwn) {
        // (the same fused multiply-add as in the pass that owns queries: every pass sees the same P, bit for bit)
        shift = HAS_PAD ? __builtin_fmaf(own_pad, kLog2eB, -row_a[r]) : -row_a[r];
        if constexpr (kNeedT2) delta_r = row_b[r];
      } else if constexpr (HAS_PAD) {
        shift = __builtin_fmaf(fmaxf(row_a[r], kMaskFloor), kLog2eB, -own_lse);
      } else {
        shift = -own_lse;
      }
      float p = __builtin_amdgcn_exp2f(__builtin_fmaf(t1[r], a.scale_log2e, shift));
      if constexpr (MASKED) {
        const int other = t * kSchedTile + rr;
        const bool visible = kKeysOwn ? own <= other && (!HAS_WINDOW || other - window < own)
                                      : other <= own && (!HAS_WINDOW || other > own - window);
        p = visible ? p : 0.f;
      }
      float grad = t2[r];
      float kept = p; // the probability the values met (the combined pass keeps it beside dS)
      if constexpr (DROP) {
        const bool keep = kKeysOwn ? ((keep_words[r >> 2][r & 3] >> col) & 1u) != 0
                                   : ((keep_bits >> (8 * (r >> 2) + (r & 3))) & 1u) != 0;
        grad = keep ? grad * a.drop.keep_scale : 0.f;
        if constexpr (!kNeedT2) p = keep ? p : 0.f;
        if constexpr (kKeepP) kept = keep ? p : 0.f;
      }
      if constexpr (kNeedT2) p *= grad - delta_r;
      t1[r] = p;
      asm volatile("" : "+v"(t1[r])); // (keeps the computation in its slice)
      if constexpr (kKeepP) {
        t2[r] = kept;
        asm volatile("" : "+v"(t2[r]));
      }
    }
    if (n == slices - 1) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[u][i] = static_cast<T>(t1[8 * u + i]);
      if constexpr (kKeepP) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 8; ++i) x2[u][i] = static_cast<T>(t2[8 * u + i]);
      }
    }
  };
  // The wave's tiles of the store: query tile own0 / 32 + wave, key tile t. A
  // tile that lies wholly above the diagonal has no place there (and holds zeros).
  unsigned char *tile_row = nullptr;
  const int own_tile = own0 / 32 + wave;
  if constexpr (STORE)
    tile_row = a.tiles + ((int64_t)(bh - a.bh0) * a.head_tiles + (int64_t)own_tile * (own_tile + 1) / 2) * kStoredPairBytes +
               lane * 16;
  auto store_tiles = [&](const Frag (&ds)[2], const Frag (&pk)[2]) __attribute__((always_inline)) {
    if constexpr (STORE) {
      if (t <= own_tile) {
        unsigned char *at = tile_row + (int64_t)t * kStoredPairBytes;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          // (written once and read once by the next pass: non-temporal, so that K and V stay in the caches)
          __builtin_nontemporal_store(pk[u], reinterpret_cast<Frag *>(at + 1024 * u));
          __builtin_nontemporal_store(ds[u], reinterpret_cast<Frag *>(at + kStoredTileBytes + 1024 * u));
        }
      }
    }
  };
  constexpr int kStoresPerTile = STORE ? 4 : 0;

  // A tile as one straight run of code between fences: the products of T1 with
  // the next tiles' loads between them, those of T2, then the accumulating
  // products of the previous tile with this tile's elementwise work between
  // them. Operands are read from LDS kRing products ahead.
  auto scheduled_tile = [&]<bool MASKED>() __attribute__((always_inline)) {
    constexpr int kRing = 4;
    constexpr int kProducts = 2 * kBlocksD;
    // the combined pass: the products of dV^T (dO^T x P) first, then those of dK^T (Q^T x dS)
    constexpr int kAccProducts = (kTwoAcc ? 2 : 1) * kProducts;
    constexpr int kOperands = kSteps + (kNeedT2 ? kSteps : 0) + kAccProducts;
    constexpr int kPerStep = (kItems + kSteps - 1) / kSteps;
    const T *b1 = o1_lds + buffer_of(0) * kTile, *b2 = o2_lds + buffer_of(0) * kTile;
    const T *bt = transposed_tile(-1);
    const T *bt2 = transposed_tile2(-1);
    Frag ring[kRing];
    auto read_operand = [&](int p) __attribute__((always_inline)) {
      if (p < kSteps) ring[p % kRing] = read_natural(b1, p);
      else if (kNeedT2 && p < 2 * kSteps) ring[p % kRing] = read_natural(b2, p - kSteps);
      else {
        const int q = p - (kNeedT2 ? 2 : 1) * kSteps;
        if (kTwoAcc && q < kProducts) ring[p % kRing] = read_transposed(bt2, q);
        else ring[p % kRing] = read_transposed(bt, q - (kTwoAcc ? kProducts : 0));
      }
    };
#pragma unroll
    for (int p = 0; p < kRing; ++p) read_operand(p);
    __builtin_amdgcn_sched_barrier(0);
    f32x16 t1, t2;
#pragma unroll
    for (int r = 0; r < 16; ++r) t1[r] = t2[r] = 0.f;
    int p = 0;
#pragma unroll
    for (int s = 0; s < kSteps; ++s, ++p) {
      t1 = Op::run(ring[p % kRing], own1[s], t1);
      if (p + kRing < kOperands) read_operand(p + kRing);
#pragma unroll
      for (int it = s * kPerStep; it < (s + 1) * kPerStep && it < kItems; ++it) stage_item(it);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (kNeedT2) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s, ++p) {
        t2 = Op::run(ring[p % kRing], own2[s], t2);
        if (p + kRing < kOperands) read_operand(p + kRing);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    Frag xn[2], xpn[2];
#pragma unroll
    for (int r = 0; r < kAhead; ++r) read_row_values(r);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < kAccProducts; ++n, ++p) {
      if (kTwoAcc && n < kProducts) {
        acc2[n % kBlocksD] = Op::run(ring[p % kRing], xp[n / kBlocksD], acc2[n % kBlocksD]);
      } else {
        const int m = n - (kTwoAcc ? kProducts : 0);
        acc[m % kBlocksD] = Op::run(ring[p % kRing], xf[m / kBlocksD], acc[m % kBlocksD]);
      }
      if (p + kRing < kOperands) read_operand(p + kRing);
      elementwise.template operator()<MASKED>(t1, t2, n, kAccProducts, xn, xpn);
      __builtin_amdgcn_sched_barrier(0);
    }
    xf[0] = xn[0], xf[1] = xn[1];
    if constexpr (kKeepP) xp[0] = xpn[0], xp[1] = xpn[1];
    store_tiles(xf, xp);
  };
  // each kind of tile in a loop of its own
  auto run_tiles = [&]<bool MASKED>(int end) __attribute__((always_inline)) {
    for (; t < end; ++t) {
      // (Vector-memory operations are counted in order. Behind the loads of tile t
      // come the stores of tile t - 2, the loads of tile t + 1 and the stores of
      // tile t - 1: none of them is waited for here. A store into the tile store
      // takes long to be acknowledged; waited for a tile after it was issued, the
      // stores cost this pass 100 us of 600.)
      if (!STORE) wait_vm<kLoadsPerTile>();
      else if (t - 1 > own_tile) wait_vm<kLoadsPerTile>(); // (a wave past its diagonal stored nothing)
      else if (t - 2 < first_tile) wait_vm<kLoadsPerTile + kStoresPerTile>(); // (the block's second tile)
      else wait_vm<kLoadsPerTile + 2 * kStoresPerTile>();
      __syncthreads(); // tile t is in LDS; the buffer written next (tile t - 2's) has been read
      scheduled_tile.template operator()<MASKED>();
    }
  };
  // delta = sum_d dO O of the lane's query, eight features at a time, then the halves of the wave and the
  // steps pair by pair. O is taken with what its rounding left out: delta stands against dP in
  // every dS of the row, and where the probabilities are concentrated (a window of a few keys, the first
  // tokens of a sequence) the rounding of O alone doubled the error of dQ and dK (bf16, a window of 2:
  // 0.0039 of their norm instead of 0.0025).
  auto finish_delta = [&]() __attribute__((always_inline)) {
    if constexpr (kOwnDelta) {
      float part[kSteps];
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          x = __builtin_fmaf(static_cast<float>(own_o[s][i]) + static_cast<float>(own_low[s][i]), static_cast<float>(own2[s][i]), x);
        part[s] = halves_sum(x);
      }
#pragma unroll
      for (int step = 1; step < kSteps; step *= 2)
#pragma unroll
        for (int s = 0; s < kSteps; s += 2 * step) part[s] += part[s + step];
      own_delta = part[0];
      if (own < S && half == 0) a.delta_out[stat_row + own] = own_delta;
    }
  };
  // The walk over the tiles of one head of the other kind.
  auto walk = [&]() __attribute__((always_inline)) {
    // prologue: the first two tiles on their way
#pragma unroll
    for (int rep = 0; rep < 2; ++rep) {
      t = first_tile - 2 + rep; // (an item loads tile t + 2)
#pragma unroll
      for (int it = 0; it < kItems; ++it) stage_item(it);
    }
    t = first_tile;
    finish_delta();

    // the block's first tile: nothing to accumulate yet; plain order
    {
      wait_vm<kLoadsPerTile>();
      __syncthreads();
#pragma unroll
      for (int it = 0; it < kItems; ++it) stage_item(it);
      f32x16 t1, t2;
#pragma unroll
      for (int r = 0; r < 16; ++r) t1[r] = t2[r] = 0.f;
      const T *b1 = o1_lds + buffer_of(0) * kTile, *b2 = o2_lds + buffer_of(0) * kTile;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) t1 = Op::run(read_natural(b1, s), own1[s], t1);
      if constexpr (kNeedT2) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) t2 = Op::run(read_natural(b2, s), own2[s], t2);
      }
#pragma unroll
      for (int r = 0; r < kAhead; ++r) read_row_values(r);
      elementwise.template operator()<true>(t1, t2, 0, 1, xf, xp);
      store_tiles(xf, xp);
      ++t;
    }

    if constexpr (kKeysOwn || HAS_WINDOW) run_tiles.template operator()<true>(masked_until);
    run_tiles.template operator()<false>(plain_until);
    if constexpr (!kKeysOwn || HAS_WINDOW) run_tiles.template operator()<true>(tiles);
    // the last tile's accumulating products
    wait_vm<0>(); // (nothing may still be on its way into LDS when the block ends)
    __syncthreads();
    {
      const T *bt = transposed_tile(-1);
      if constexpr (kTwoAcc) {
        const T *bt2 = transposed_tile2(-1);
#pragma unroll
        for (int n = 0; n < 2 * kBlocksD; ++n)
          acc2[n % kBlocksD] = Op::run(read_transposed(bt2, n), xp[n / kBlocksD], acc2[n % kBlocksD]);
      }
#pragma unroll
      for (int n = 0; n < 2 * kBlocksD; ++n)
        acc[n % kBlocksD] = Op::run(read_transposed(bt, n), xf[n / kBlocksD], acc[n % kBlocksD]);
    }
  };
  if constexpr (PACKED && kKeysOwn) {
#pragma unroll 1
    for (int g = 0; g < group_heads; ++g) {
      if (g > 0) __syncthreads(); // every wave has read its last operands: the buffers may be written again
      start_sources(o1_p + g * st_o1.h, o2_p + g * st_o2.h, stat_row + g * stat_step);
      walk();
    }
  } else {
    start_sources(o1_p, o2_p, stat_row);
    walk();
  }

  // PACKED: the gradients leave through the wave's part of LDS, in whole rows. (Straight from the accumulators a
  // store is 16 bytes of 32 rows, and the blocks of short walks, which a window makes, sent two thirds of
  // the cache's requests that way.)
  if constexpr (PACKED) __syncthreads(); // every wave has read its last operands
  else if (own >= S) return;
  typedef T Out4 __attribute__((ext_vector_type(4)));
  auto store = [&](const f32x16 (&sums)[kBlocksD], void *out_base, const Strides3 &st_out, float factor)
                   __attribute__((always_inline)) {
    if constexpr (PACKED && kKeysOwn) {
      if (part_slot >= 0) {
        if (own >= S) return;
        float *fp = a.partial + ((part_slot * 2 + (out_base == a.dv ? 1 : 0)) * kOwnPerBlock + 32 * wave + col) * (int64_t)D;
#pragma unroll
        for (int i = 0; i < kBlocksD; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<float4 *>(fp + 32 * i + 8 * j + 4 * half) =
                make_float4(sums[i][4 * j] * factor, sums[i][4 * j + 1] * factor, sums[i][4 * j + 2] * factor,
                            sums[i][4 * j + 3] * factor);
        return;
      }
    }
    if constexpr (PACKED) {
      constexpr int kRow = D + 8, kRowLanes = D / 8; // (rows 16 bytes apart in the banks)
      static_assert(4 * 32 * kRow <= 2 * kSchedBuffers * kTile, "the tiles' place holds the four waves' rows");
      T *const mine = o1_lds + wave * (32 * kRow);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront"); // (the rows of the gradient before have been read)
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = 0; i < kBlocksD; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          Out4 w;
#pragma unroll
          for (int tt = 0; tt < 4; ++tt) w[tt] = static_cast<T>(sums[i][4 * j + tt] * factor);
          *reinterpret_cast<Out4 *>(mine + col * kRow + 32 * i + 8 * j + 4 * half) = w;
        }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      T *const rows = static_cast<T *>(out_base) + (kKeysOwn ? kv_hd : hd) * st_out.h + (start + wave_own0) * st_out.s;
#pragma unroll
      for (int r0 = 0; r0 < 32; r0 += kWave / kRowLanes) {
        const int r = r0 + lane / kRowLanes, at = 8 * (lane % kRowLanes);
        const Frag w = *reinterpret_cast<const Frag *>(mine + r * kRow + at);
        if (wave_own0 + r < S) *reinterpret_cast<Frag *>(rows + r * st_out.s + at) = w;
      }
      return;
    }
    T *op = static_cast<T *>(out_base) + b * st_out.b + (kKeysOwn ? kv_hd : hd) * st_out.h + (start + own) * st_out.s;
#pragma unroll
    for (int i = 0; i < kBlocksD; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        Out4 w;
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) w[tt] = static_cast<T>(sums[i][4 * j + tt] * factor);
        *reinterpret_cast<Out4 *>(op + 32 * i + 8 * j + 4 * half) = w;
      }
  };
  const float p_factor = DROP ? a.drop.keep_scale : 1.0f; // the 1/(1-p) of the kept probabilities
  if constexpr (ROLE == kRoleDQ) store(acc, a.dq, a.sdq, a.scale);
  else if constexpr (ROLE == kRoleDK) store(acc, a.dk, a.sdk, a.scale);
  else if constexpr (ROLE == kRoleDV) store(acc, a.dv, a.sdv, p_factor);
  else {
    store(acc, a.dk, a.sdk, a.scale);
    store(acc2, a.dv, a.sdv, p_factor);
  }
}

// delta[bh, q] = sum_d dO[q, d] * O[q, d], fp32. D / 8 lanes share a row.
template <typename T, int D>
__global__ __launch_bounds__(kBlockThreads) void attention_delta_kernel(
    float *delta, const T *out, const T *dout, Strides3 so, Strides3 sdo, int S,
    int heads, int64_t rows) {
  constexpr int kLanes = D / 8;
  constexpr int kRows = kBlockThreads / kLanes;
  int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / kLanes;
  const bool live = row < rows;
  if (!live) row = rows - 1; // the lanes of a group stay together for the reduction
  const int part = threadIdx.x % kLanes;
  const int64_t bh = row / S;
  const int q = (int)(row - bh * S);
  const int64_t b = bh / heads, hd = bh - b * heads;
  typedef T Vec8 __attribute__((ext_vector_type(8)));
  const Vec8 o = *reinterpret_cast<const Vec8 *>(out + b * so.b + hd * so.h + (int64_t)q * so.s + 8 * part);
  const Vec8 g = *reinterpret_cast<const Vec8 *>(dout + b * sdo.b + hd * sdo.h + (int64_t)q * sdo.s + 8 * part);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s = __builtin_fmaf(static_cast<float>(o[i]), static_cast<float>(g[i]), s);
  s = sum_over_lanes<kLanes>(s);
  if (live && part == 0) delta[row] = s;
}

} // namespace
} // namespace oslo
