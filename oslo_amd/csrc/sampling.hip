// Draws one token per row of logits from given uniform numbers, after
// temperature, top-k, top-p and min-p. With x = logit / temperature and the
// order "larger logit first, lower index first among equals":
//   K1 = the first top_k tokens of that order (0: all),
//   K2 = the shortest run of K1 from its front with mass >= top_p * mass(K1),
//        mass(j) = exp(x_j - max x),
//   K3 = the tokens of K2 with mass >= min_p,
//   token = the first index, in index order, at which the running mass over K3
//           exceeds u * mass(K3).
// The kept set is a front of the order whatever the settings, so it is described by
// the logit it ends at and by how many of the tokens with exactly that logit are in.
//
// Which token comes out is a whole number, so a border of the filters or of the
// draw must not move with the order of a sum. Masses are therefore whole numbers
// too: exp in 64 bits, times 2^S, rounded (S = 61 - ceil(log2 vocabulary), at most 49; 45 at
// fifty thousand tokens; a rounding of 2^-46 of the largest mass, ten million
// times finer than a 32-bit sum). Sums of whole numbers are exact in any order:
// histograms may use atomics and every run gives the same token.
//
// One block takes a row, 1024 threads and a CU for itself up to 256 rows; beyond that
// 512, two to a CU, one waiting for memory or at a barrier while the other computes
// (1000 rows of 50257 fp32 logits with top-p: 118 against 130 us). It holds the row in
// registers and LDS (53248 logits of 32 bits, or 20480, twice that in 16 bits; what exceeds them
// is read again, ahead of its use), each wave a run of it. Such a row is read in 5 to 8 us; what
// costs the time then is arithmetic, one operation in 64 bits after another, and
// barriers (one row of 1024 threads, thousands of cycles: reading 10, the count below 12, its
// border 3.5, the exact pass 30, the border in the window 5 to 7, the draw 5.5):
//  - top-k goes first: a histogram of the threads' own maxima gives a bound that
//    at least k logits reach and few exceed. They go into a list in LDS, which is all
//    the rest looks at; up to 512 of them are ranked by counting, without a sort.
//  - top-p over a whole row: the logits are counted over 2048 steps of the distance to
//    the largest one. Masses inside a step differ by 0.9 %, so the counts place the border
//    of a share p to 0.9 % p (1 - p) of the mass, a step or a few. The one exact pass
//    then sums all masses, sums those in front of that window by waves, and
//    lists the logits in the window; the exact sums say whether the border really is among the listed ones
//    (else an exact search finds it: the hint never decides). The listed ones' masses are summed over
//    finer steps, and the few in the step of the border are ranked (all of them ranked
//    by counting took 34 thousand cycles, this 5 to 7).
//  - the draw finds the wave in whose run the running mass passes its target, its
//    chunk, which all waves sum together, and looks inside that.
// Windows too full for the list (equal logits by the thousand) are searched by
// histograms over the bits of the logits. Measured, us a call: one row of 50257 fp32 logits, top-k 50 and
// top-p, 12.1; 256 rows in bf16, settings of their own, 35; 1000 rows in fp32, top-p 0.92, 118 captured, 125 eager, 132
// under the profiler, which counts 475 MB read, 2.4 times the logits: what a row has beyond the 20480 that are held comes
// again for the maximum, the count and the exact pass, at 3.8 TB/s on average next to some sixty vector
// instructions a logit, many of them in 64 bits.

#include "common.hpp"

namespace oslo {
namespace {

constexpr int kBins = 2048;
constexpr int kMostWaves = 16;

typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned long long u64;

// A setting of the call: one number, or one per row.
template <typename V>
struct Setting {
  const V *rows;
  double all;
  __device__ __forceinline__ double at(int64_t row) const { return rows ? (double)rows[row] : all; }
};

struct SampleArgs {
  int64_t *tokens;
  float *logprobs; // or null
  const void *logits;
  int64_t row_stride;
  const float *uniforms;
  Setting<float> temperature, top_p, min_p;
  Setting<int> top_k;
  int vocab, mass_bits;
};

// Whole numbers in the order of the floats (NaN is taken as -inf before).
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t key) {
  return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// 2^((i - 1/2) / 1024), i = 0 .. 1023, by the Taylor series of the exponential (to the
// eighteenth power: below 2^-60 of the result); once per block.
constexpr int kTable = 1024;
constexpr double kStep = 0.69314718055994530942 / kTable; // of the natural logarithm between two entries
__device__ __forceinline__ double table_entry(int i) {
  const double z = ((double)i - 0.5) * kStep;
  double s = 1.0;
#pragma unroll
  for (int n = 18; n >= 1; --n) s = __builtin_fma(s * z, 1.0 / n, 1.0);
  return s;
}

// The largest float below x (x > next_below(y) just where x >= y); -inf stays.
__device__ __forceinline__ float next_below(float x) {
  if (x == -INFINITY) return x;
  return key_value((x == 0.f ? 0x7fffffffu : order_key(x)) - 1); // (0 and -0 are one number)
}
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ u64 dpp_u64(u64 v) { // (lanes that receive nothing get 0)
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, true);
  return (u64)hi << 32 | lo;
}
// Sum over the lanes up to and including this one: within rows of 16 by shifts of 1, 2,
// 4 and 8, then the last lane of a row to the next row, and lane 31 to the upper half.
__device__ __forceinline__ u64 wave_scan_u64(u64 v) {
  v += dpp_u64<0x111>(v);
  v += dpp_u64<0x112>(v);
  v += dpp_u64<0x114>(v);
  v += dpp_u64<0x118>(v);
  v += dpp_u64<0x142, 0xa>(v);
  v += dpp_u64<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ u64 lane_u64(u64 v, int lane) { // (of a lane that is the same for all)
  return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
// Sum over the wave, for every lane: rows of 16 on the vector ALU, the four rows by lane reads.
__device__ __forceinline__ u64 wave_sum_u64(u64 v) {
  v += dpp_u64<0xB1>(v);
  v += dpp_u64<0x4E>(v);
  v += dpp_u64<0x141>(v);
  v += dpp_u64<0x140>(v);
  u64 sum = 0;
#pragma unroll
  for (int r = 0; r < 4; ++r)
    sum += (u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), 16 * r) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, 16 * r);
  return sum;
}

constexpr int kListed = 2048; // logits the list in LDS holds
constexpr int kRanked = 512;  // ... of which so many are ranked by counting

struct alignas(16) SampleLds {
  u64 bins[kBins];
  union {
    u64 list[kListed]; // order_key(logit) << 32 | ~index: distinct, and in the filters' order
    uint32_t counts[kBins + kWave];
  };
  u64 picked[kRanked], ranked[kRanked];
  double table[kTable];
  u64 wave_sums[kMostWaves], wave_all[kMostWaves], wave_kept[kMostWaves];
  float wave_max[kMostWaves], wave_min[kMostWaves];
  u64 found_before, found_value; // results of a search, written by the one thread that finds them
  double log_total;
  int found_at, found_too;
  int listed, num_picked;
  uint32_t bound;
};
__device__ __forceinline__ u64 list_entry(float x, int index) {
  return (u64)order_key(x) << 32 | (uint32_t)~index;
}
__device__ __forceinline__ float entry_logit(u64 e) { return key_value((uint32_t)(e >> 32)); }
__device__ __forceinline__ int entry_index(u64 e) { return (int)~(uint32_t)e; }

// A running sum over kBins values: each thread's share (consecutive ones), what lies
// before it, and the total.
template <int kThreads>
struct BinScan {
  static constexpr int kEach = kBins / kThreads;
  u64 v[kEach], before, mine, total;
  __device__ __forceinline__ static int bin(int i) { return (int)threadIdx.x * kEach + i; }
};
template <int kThreads>
__device__ __forceinline__ BinScan<kThreads> scan_values(SampleLds &lds, BinScan<kThreads> s) {
  constexpr int kBinsEach = s.kEach, kWaves = kThreads / kWave;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  s.mine = 0;
#pragma unroll
  for (int i = 0; i < kBinsEach; ++i) s.mine += s.v[i];
  const u64 upto = wave_scan_u64(s.mine);
  if (lane == kWave - 1) lds.wave_sums[wave] = upto;
  __syncthreads();
  const u64 waves = wave_scan_u64(lane < kWaves ? lds.wave_sums[lane] : 0);
  s.before = upto - s.mine + (wave > 0 ? lane_u64(waves, wave - 1) : 0);
  s.total = lane_u64(waves, kWaves - 1);
  return s;
}
// The bins must be complete (a barrier has passed).
template <int kThreads>
__device__ __forceinline__ BinScan<kThreads> scan_bins(SampleLds &lds) {
  BinScan<kThreads> s;
#pragma unroll
  for (int i = 0; i < s.kEach; ++i) s.v[i] = lds.bins[s.bin(i)];
  return scan_values(lds, s);
}
// f(bin, sum before it, its value) for the first bin at which the running sum reaches
// `target` (0 < target <= total), by the one thread that has it.
template <int kThreads, typename F>
__device__ __forceinline__ void at_target(const BinScan<kThreads> &s, u64 target, F &&f) {
  u64 run = s.before;
  if (run < target && run + s.mine >= target) {
#pragma unroll
    for (int i = 0; i < s.kEach; ++i) {
      if (run < target && run + s.v[i] >= target) f(s.bin(i), run, s.v[i]);
      run += s.v[i];
    }
  }
}
// The same, for every thread.
struct Found {
  int at;
  u64 before, value;
};
template <int kThreads>
__device__ __forceinline__ Found find_bin(SampleLds &lds, const BinScan<kThreads> &s, u64 target) {
  at_target(s, target, [&](int at, u64 before, u64 value) __attribute__((always_inline)) {
    lds.found_at = at;
    lds.found_before = before;
    lds.found_value = value;
  });
  __syncthreads();
  Found f;
  f.at = lds.found_at, f.before = lds.found_before, f.value = lds.found_value;
  __syncthreads(); // (the bins and the results may be written again)
  return f;
}

// A row is cut into pieces of 16 bytes, and each wave takes a run of them, chunk by
// chunk of 64. Chunks that the registers hold, and the most that LDS holds behind
// them (with the tables above, 145 of a CU's 160 KiB).
constexpr int kInRegisters = 7;
constexpr int most_in_lds(int threads) { return threads == 1024 ? 6 : 3; }

template <typename T, int kThreads>
__global__ __launch_bounds__(kThreads, 4) void sample_kernel(const SampleArgs a) {
  constexpr int kWaves = kThreads / kWave, kMostInLds = most_in_lds(kThreads), kBinsEach = kBins / kThreads;
  constexpr int kVec = Io<T>::kVec; // logits of a 16-byte load
  using V = RawVec<T, kVec>;
  extern __shared__ __align__(16) unsigned char lds_raw[];
  SampleLds &lds = *reinterpret_cast<SampleLds *>(lds_raw);
  V *const lds_held = reinterpret_cast<V *>(lds_raw + sizeof(SampleLds)); // [chunk - kInRegisters][thread]
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int64_t row = blockIdx.x;
  const int vocab = a.vocab;
  const T *const logits = static_cast<const T *>(a.logits) + row * a.row_stride;
  // Rows of an odd number of logits begin anywhere. They are read in the aligned
  // 16-byte pieces that hold any of them: the row begins `lead` logits into the first
  // piece (the logits beside the row's in its first and last piece are masked).
  const int lead = (int)((reinterpret_cast<uintptr_t>(logits) & 15u) / sizeof(T));
  const V *const pieces = reinterpret_cast<const V *>(logits - lead);
  const int last_piece = (vocab + lead - 1) / kVec;
  const int chunks = last_piece / kThreads + 1; // ... of a wave
  const T kNothing = static_cast<T>(-INFINITY);
  bool infinite = false; // the largest logit is +inf: only those count, as zeros among -inf
  // the piece that lane `l` of this wave holds of chunk c, and the index of its first logit (may be negative)
  auto piece_of = [&](int c, int l) __attribute__((always_inline)) { return (wave * chunks + c) * kWave + l; };
  auto first_in = [&](int piece) __attribute__((always_inline)) { return piece * kVec - lead; };
  auto first_of = [&](int c, int l) __attribute__((always_inline)) { return first_in(piece_of(c, l)); };
  auto load_raw = [&](int piece) __attribute__((always_inline)) {
    return pieces[piece < last_piece ? piece : last_piece]; // (no branch: the loads of a thread are issued together)
  };
  // Beside the row: -inf. NaN becomes -inf, -0 becomes 0 (they are equal logits).
  auto clean = [&](V &v, int piece) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) v[e] = static_cast<T>(fmaxf(static_cast<float>(v[e]) + 0.f, -INFINITY));
    const int first = __builtin_amdgcn_readfirstlane(piece); // (the wave's pieces lie one behind the other)
    if (first == 0 || first + kWave > last_piece)
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[e] = (unsigned)(first_in(piece) + e) < (unsigned)vocab ? v[e] : kNothing;
  };
  auto only_infinite = [&](V &v) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) v[e] = static_cast<float>(v[e]) == INFINITY ? static_cast<T>(0.f) : kNothing;
  };
  auto load = [&](int piece) __attribute__((always_inline)) {
    V v = load_raw(piece);
    clean(v, piece);
    if (infinite) only_infinite(v);
    return v;
  };
  V held[kInRegisters];
  const int in_lds = chunks - kInRegisters < kMostInLds ? chunks - kInRegisters : kMostInLds;
#pragma unroll
  for (int c = 0; c < kInRegisters; ++c) held[c] = load_raw(piece_of(c, lane));
  if (in_lds > 0) {
    V more[kMostInLds];
#pragma unroll
    for (int c = 0; c < kMostInLds; ++c) more[c] = load_raw(piece_of(kInRegisters + c, lane));
#pragma unroll
    for (int c = 0; c < kMostInLds; ++c)
      if (c < in_lds) {
        clean(more[c], piece_of(kInRegisters + c, lane));
        lds_held[c * kThreads + tid] = more[c];
      }
  }
#pragma unroll
  for (int c = 0; c < kInRegisters; ++c) clean(held[c], piece_of(c, lane));
#pragma unroll 1
  for (int i = tid; i < kTable; i += kThreads) lds.table[i] = table_entry(i);
#pragma unroll
  for (int b = 0; b < kBinsEach; ++b) lds.bins[tid + b * kThreads] = 0;
  if (tid == 0) lds.listed = 0;
  // f(chunk, vector) for every vector of this thread. The empty statement "changes"
  // the vector: without it the compiler works out ahead, for all chunks at once, what
  // several passes have in common (conversions, whole masses, indices), and spills it.
  int at_lane = lane; // the lane, for the indices of the vector being visited
  auto for_chunks = [&](auto &&f) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < kInRegisters; ++c)
      if (c < chunks) {
        u32x4_t w = __builtin_bit_cast(u32x4_t, held[c]);
        at_lane = lane;
        asm volatile("" : "+v"(w), "+v"(at_lane));
        f(c, __builtin_bit_cast(V, w));
        __builtin_amdgcn_sched_barrier(0);
      }
    at_lane = lane;
    // (what is read again is on its way while the chunk before it is worked on)
    V ahead{};
    if (chunks > kInRegisters + kMostInLds) ahead = load_raw(piece_of(kInRegisters + kMostInLds, lane));
#pragma unroll 1
    for (int c = kInRegisters; c < chunks; ++c) {
      V v;
      if (c < kInRegisters + kMostInLds) {
        v = lds_held[(c - kInRegisters) * kThreads + tid];
      } else {
        v = ahead;
        ahead = load_raw(piece_of(c + 1, lane));
        clean(v, piece_of(c, lane));
        if (infinite) only_infinite(v);
      }
      f(c, v);
    }
  };
  // the same, all of it read again (for searches that hardly ever run: little code)
  auto for_chunks_again = [&](auto &&f) __attribute__((always_inline)) {
#pragma unroll 1
    for (int c = 0; c < chunks; ++c) f(c, load(piece_of(c, lane)));
  };

  // the largest logit of the thread, then of the row
  float mine = -INFINITY;
  for_chunks([&](int, const V &v) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) mine = fmaxf(mine, static_cast<float>(v[e]));
  });
  float top = wave_allreduce(mine, OpMax());
  float low = -wave_allreduce(mine == -INFINITY ? -INFINITY : -mine, OpMax()); // smallest finite maximum
  if (lane == 0) lds.wave_max[wave] = top, lds.wave_min[wave] = low;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = fmaxf(top, lds.wave_max[w]), low = fminf(low, lds.wave_min[w]);
  if (top == -INFINITY) { // nothing can be drawn
    if (tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
    return;
  }
  if (top == INFINITY) {
    infinite = true;
    mine = mine == INFINITY ? 0.f : -INFINITY;
    top = low = 0.f;
#pragma unroll
    for (int c = 0; c < kInRegisters; ++c) only_infinite(held[c]);
    for (int c = 0; c < in_lds; ++c) only_infinite(lds_held[c * kThreads + tid]);
  }

  const double temperature = a.temperature.at(row);
  const double k_setting = a.top_k.at(row);
  if (!(temperature > 0.0) || k_setting == 1.0) { // the first of the largest
    if (tid == 0) lds.found_at = vocab;
    __syncthreads();
    if (mine == top)
      for_chunks_again([&](int c, const V &v) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < kVec; ++e)
          if (static_cast<float>(v[e]) == top) atomicMin(&lds.found_at, first_of(c, lane) + e);
      });
    __syncthreads();
    if (tid == 0) {
      a.tokens[row] = lds.found_at;
      if (a.logprobs) a.logprobs[row] = 0.f;
    }
    return;
  }

  // Mass of a logit relative to the largest one's, as a whole number of 2^-S: with
  // z = 1024 log2(e) (top - x) / temperature = n + r, 0 <= r < 1, it is 2^(-n / 1024)
  // from the table times e^-(r kStep), a polynomial of the third power about r = 1/2 (the
  // next term is below 2^-50). The result times 2^S is below 2^52: adding 2^52 rounds it to a
  // whole number, in the low bits.
  const double per_unit = 1.4426950408889634074 / temperature;
  const double per_entry = per_unit * kTable;
  constexpr double kRounding = 4503599627370496.0;
  constexpr u64 kMassBits = 0xfffffffffffffull;
  // Of several logits at once, so that one's table read and its chain of 64-bit
  // operations hide behind the others': w[i] = mass + 2^52.
  auto rounded_masses = [&]<int N>(const float (&x)[N], double (&w)[N]) __attribute__((always_inline)) {
    constexpr double d = kStep, h = kStep / 2;
    double r[N];
    int n[N];
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = fmin(((double)top - (double)x[i]) * per_entry, 960.0 * kTable); // (a mass of 0)
#pragma unroll
    for (int i = 0; i < N; ++i) n[i] = (int)-r[i]; // (towards zero)
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = lds.table[n[i] & (kTable - 1)];
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = __builtin_amdgcn_fract(r[i]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      double p = __builtin_fma(r[i], -(d * d * d) / 6.0, d * d / 2.0 * (1.0 + h));
      p = __builtin_fma(p, r[i], -d * (1.0 + h + h * h / 2.0));
      r[i] = __builtin_fma(p, r[i], 1.0 + h + h * h / 2.0 + h * h * h / 6.0);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = __builtin_ldexp(r[i] * w[i], (n[i] >> 10) + a.mass_bits) + kRounding;
  };
  auto units_of = [&](float x) __attribute__((always_inline)) -> u64 {
    double w[1];
    rounded_masses({x}, w);
    return __builtin_bit_cast(u64, w[0]) & kMassBits;
  };
  // Steps of the distance to the largest logit, falling as x rises.
  auto step_of = [&](float x, float per_step) __attribute__((always_inline)) -> int {
    return (int)fminf((top - x) * per_step, (float)(kBins - 1));
  };

  // The kept front of the order: logits above `cut`, and those equal to it with an
  // index up to `cut_index`; of those the ones not below `floor_x` (min-p).
  float cut = -INFINITY, floor_x = -INFINITY;
  int cut_index = -1;
  bool cutting = false; // (there is a cut at all)
  auto in_front = [&](float x, int index) __attribute__((always_inline)) {
    return (x > cut) | ((x == cut) & (index <= cut_index)); // (no branch)
  };
  const double min_mass = a.min_p.at(row);
  if (min_mass > 0.0) {
    // mass >= min_p where the logit reaches top + temperature * ln(min_p); the largest always stays
    const double least = (double)top + (min_mass < 1.0 ? log(min_mass) * temperature : 0.0);
    floor_x = (float)least;
    if ((double)floor_x < least) floor_x = key_value(order_key(floor_x) + 1);
  }
  const double p_setting = a.top_p.at(row) < 1.0 ? fmax(a.top_p.at(row), 0.0) : 1.0; // (NaN: everything)
  double u = (double)a.uniforms[row];
  u = u >= 0.0 ? (u < 1.0 ? u : 0.99999994039535522) : 0.0;
  // the target of top-p among `total` units, and of the draw
  auto share_of = [&](u64 total) __attribute__((always_inline)) -> u64 {
    const double wanted = __builtin_ceil(p_setting * (double)total);
    const u64 target = wanted < 1.0 ? 1 : (u64)wanted;
    return target > total ? total : target;
  };
  auto drawn_of = [&](u64 total) __attribute__((always_inline)) -> u64 {
    const u64 target = (u64)(u * (double)total);
    return target < total ? target : total - 1;
  };
  auto log_of = [&](u64 total) __attribute__((always_inline)) { return log(__builtin_ldexp((double)total, -a.mass_bits)); };
  auto finish = [&](int token, float x, double log_total) __attribute__((always_inline)) { // (one thread)
    a.tokens[row] = token;
    if (a.logprobs) a.logprobs[row] = (float)(((double)x - (double)top) / temperature - log_total);
  };

  auto clear_bins = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < kBinsEach; ++b) lds.bins[tid + b * kThreads] = 0;
    __syncthreads();
  };
  // f(entry) for this thread's share of the list
  auto for_listed = [&](auto &&f) __attribute__((always_inline)) {
    const int n = lds.listed;
#pragma unroll 1
    for (int i = tid; i < n; i += kThreads) {
      const u64 e = lds.list[i];
      f(entry_logit(e), entry_index(e));
    }
  };
  auto all_again = [&](auto &&f) __attribute__((always_inline)) {
    for_chunks_again([&](int c, const V &v) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const float x = static_cast<float>(v[e]);
        if (x != -INFINITY) f(x, first_of(c, lane) + e);
      }
    });
  };
  auto append = [&](float x, int index) __attribute__((always_inline)) {
    const int at = atomicAdd(&lds.listed, 1);
    if (at < kListed) lds.list[at] = list_entry(x, index);
  };
  // Logits to be listed are marked, a bit each, while a pass that only compares goes over the row, and listed
  // behind it: few are (top-k 300 of 50257: 27 -> 25 us). The window's are listed where the masses are worked out,
  // where the marks' two registers made others spill.
  constexpr int kMarked = 64 / kVec; // chunks
  constexpr float kLowest = -3.40282347e38f;
  u64 marks = 0;
  auto mark = [&](int c, uint32_t bits) __attribute__((always_inline)) { marks |= (u64)bits << (c * kVec); };
  auto list_marked = [&]() __attribute__((always_inline)) {
#pragma unroll 1
    while (marks) {
      const int bit = __builtin_ctzll(marks), index = first_of(bit / kVec, lane) + bit % kVec;
      marks &= marks - 1;
      append(infinite ? 0.f : static_cast<float>(logits[index]) + 0.f, index);
    }
  };
  auto pick = [&](float x, int index) __attribute__((always_inline)) {
    const int at = atomicAdd(&lds.num_picked, 1);
    if (at < kRanked) lds.picked[at] = list_entry(x, index);
  };
  auto start_list = [&]() __attribute__((always_inline)) {
    if (tid == 0) lds.listed = 0;
    __syncthreads();
  };
  // n <= kRanked entries into lds.ranked, in order: four threads (two or one where there
  // are more than a quarter or half of the block) count the entries before one.
  auto share_for = [&](int n) __attribute__((always_inline)) {
    return n <= kThreads / 4 ? 2 : n <= kThreads / 2 ? 1 : 0;
  };
  // f(rank, entry) for each.
  auto rank_entries = [&](const u64 *entries, int n, auto &&f) __attribute__((always_inline)) {
    const int share = share_for(n), i = tid >> share;
    if (i < n) {
      const u64 e = entries[i];
      const int part = tid & ((1 << share) - 1);
      int before = 0;
#pragma unroll 8
      for (int j = part; j < n; j += 1 << share) before += entries[j] > e ? 1 : 0;
      // (threads of an entry are neighbours)
      if (share >= 1) before += __builtin_amdgcn_update_dpp(0, before, 0xB1, 0xf, 0xf, true);
      if (share == 2) before += __builtin_amdgcn_update_dpp(0, before, 0x4E, 0xf, 0xf, true);
      if (part == 0) {
        lds.ranked[before] = e;
        f(before, e);
      }
    }
    __syncthreads();
  };
  constexpr int kRankedEach = kRanked / kWave; // ranks a lane of one wave takes, one behind the other

  // Among the logits that `each` visits: the key at which the running weight reaches
  // `target`, what is missing there, and the weight of all logits with that key.
  struct Border {
    uint32_t key;
    u64 missing, value;
  };
  auto by_bits = [&](auto &&each, auto &&weight, u64 target) __attribute__((always_inline)) {
    Border r;
    r.key = 0;
    int bits = 0;
#pragma unroll 1
    for (int level = 0; level < 3; ++level) {
      const int take = level == 2 ? 10 : 11, shift = 32 - bits - take;
      const uint32_t mask = (1u << take) - 1;
      clear_bins();
      each([&](float x, int index) __attribute__((always_inline)) {
        const uint32_t k = order_key(x);
        if (bits && (k >> (32 - bits)) != r.key) return;
        const u64 w = weight(x, index);
        if (w) atomicAdd(&lds.bins[mask - ((k >> shift) & mask)], w);
      });
      __syncthreads();
      const Found f = find_bin(lds, scan_bins<kThreads>(lds), target);
      target -= f.before;
      r.key = r.key << take | (mask - (uint32_t)f.at);
      r.value = f.value;
      bits += take;
    }
    r.missing = target;
    return r;
  };
  // Of a chunk of 64 pieces, before which the running weight is `before`, the lane has the piece v with the
  // weights w: f(index, logit) where the running weight exceeds `target`, by one lane.
  auto inside_chunk = [&](const V &v, const u64 (&w)[kVec], int piece, u64 before, u64 target, auto &&f)
                          __attribute__((always_inline)) {
    u64 sum = 0;
#pragma unroll
    for (int e = 0; e < kVec; ++e) sum += w[e];
    u64 at = before + wave_scan_u64(sum) - sum;
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      if (at <= target && at + w[e] > target) f(first_in(piece) + e, static_cast<float>(v[e])); // exactly one
      at += w[e];
    }
  };
  // The index of the `ties`-th of the logits equal to x that are in the front.
  auto index_of_tie = [&](float x, u64 ties) __attribute__((always_inline)) -> int {
    auto is_tie = [&](float y, int i) __attribute__((always_inline)) -> u64 { return y == x && in_front(y, i) ? 1 : 0; };
    clear_bins();
    for_chunks_again([&](int c, const V &v) __attribute__((always_inline)) {
      u64 sum = 0;
#pragma unroll
      for (int e = 0; e < kVec; ++e) sum += is_tie(static_cast<float>(v[e]), first_of(c, lane) + e);
      sum = wave_sum_u64(sum);
      if (lane == 0) lds.bins[wave * chunks + c] = sum;
    });
    __syncthreads();
    const Found f = find_bin(lds, scan_bins<kThreads>(lds), ties);
    if (wave == 0) {
      const int piece = f.at * kWave + lane;
      const V v = load(piece);
      u64 w[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) w[e] = is_tie(static_cast<float>(v[e]), first_in(piece) + e);
      inside_chunk(v, w, piece, f.before, ties - 1,
                   [&](int index, float) __attribute__((always_inline)) { lds.found_at = index; });
    }
    __syncthreads();
    const int index = lds.found_at;
    __syncthreads();
    return index;
  };
  // The front now ends at b.key, of whose logits the first ceil(b.missing / each) are in. (All that were counted:
  // those up to the front's old end, where that lies among them.)
  auto set_cut = [&](const Border &b, u64 each) __attribute__((always_inline)) {
    const u64 ties = (b.missing + each - 1) / each;
    const float x = key_value(b.key);
    const int index = ties < b.value / each ? index_of_tie(x, ties) : cutting && x == cut ? cut_index : vocab;
    cut = x;
    cut_index = index;
    cutting = true;
  };
  auto one_each = [](float, int) __attribute__((always_inline)) -> u64 { return 1; };
  // The listed entry at which the running weight reaches `target`: entries are
  // distinct, so their 64 bits, eleven at a time from the top, lead to one (of the
  // index 19 bits can differ).
  auto entry_border = [&](auto &&weight, u64 target) __attribute__((always_inline)) -> u64 {
    u64 prefix = 0;
    int below = 64; // bits below the prefix
#pragma unroll 1
    while (below > 0) {
      const int take = below == 42 ? 10 : below == 32 ? 13 : below == 8 ? 8 : 11; // 11 11 10 | 13 that are alike, 11, 8
      if (take == 13) {
        prefix = prefix << 13 | 0x1fff;
        below -= 13;
        continue;
      }
      const u64 mask = (1u << take) - 1;
      clear_bins();
      const int n = lds.listed;
#pragma unroll 1
      for (int i = tid; i < n; i += kThreads) {
        const u64 e = lds.list[i];
        if (below < 64 && (e >> below) != prefix) continue;
        const u64 w = weight(entry_logit(e));
        if (w) atomicAdd(&lds.bins[mask - ((e >> (below - take)) & mask)], w);
      }
      __syncthreads();
      const Found f = find_bin(lds, scan_bins<kThreads>(lds), target);
      target -= f.before;
      prefix = prefix << take | (mask - (u64)f.at);
      below -= take;
    }
    return prefix;
  };
  auto cut_at = [&](u64 entry) __attribute__((always_inline)) {
    cut = entry_logit(entry);
    cut_index = entry_index(entry);
    cutting = true;
  };

  if (k_setting > 1.0 && k_setting < (double)vocab) {
    const u64 k = (u64)k_setting;
    bool listed = false;
    float bound = -INFINITY;
    if (k <= kThreads) {
      // the step that the k-th largest of the threads' maxima lies in: the logits up to it are at least k
      // (the bins and the list have been cleared with the row's load)
      const float per_step = top > low ? fminf((float)(kBins - 1) / (top - low), 1.0e30f) : 0.f;
      if (mine != -INFINITY) atomicAdd(&lds.bins[step_of(mine, per_step)], (u64)1);
      __syncthreads();
      const BinScan<kThreads> s = scan_bins<kThreads>(lds);
      if (s.total >= k) {
        const Found f = find_bin(lds, s, k);
        // at or below the smallest number of that step: of the margin, a hundredth is for the product's rounding,
        // the next number below for the difference's
        // (a finite number: what lies beside the row is -inf, and has no place to be read from)
        bound = fmaxf(per_step > 0.f ? next_below(top - ((float)f.at + 1.01f) / per_step) : low, kLowest);
        for_chunks([&](int c, const V &v) __attribute__((always_inline)) {
          if (c < kMarked) {
            uint32_t bits = 0;
#pragma unroll
            for (int e = 0; e < kVec; ++e) bits |= static_cast<float>(v[e]) >= bound ? 1u << e : 0u;
            mark(c, bits);
          } else {
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
              const float x = static_cast<float>(v[e]);
              if (x >= bound) append(x, first_of(c, at_lane) + e);
            }
          }
        });
        list_marked();
        __syncthreads();
        listed = lds.listed <= kListed;
      }
      __syncthreads();
    }
    const u64 *entries = lds.list;
    int num_entries = lds.listed;
    if (listed && num_entries > kRanked && k <= kRanked) {
      // too many to rank: those in finer steps between the bound and the largest, up to the step of the k-th
      const float range = top - bound;
      const float per_bin = range > 0.f ? fminf((float)(kBins - 1) / range, 1.0e30f) : 0.f;
      if (tid == 0) lds.num_picked = 0;
      clear_bins();
      for_listed([&](float x, int) __attribute__((always_inline)) { atomicAdd(&lds.bins[step_of(x, per_bin)], (u64)1); });
      __syncthreads();
      const Found f = find_bin(lds, scan_bins<kThreads>(lds), k);
      for_listed([&](float x, int i) __attribute__((always_inline)) {
        if (step_of(x, per_bin) <= f.at) pick(x, i);
      });
      __syncthreads();
      if (lds.num_picked <= kRanked) entries = lds.picked, num_entries = lds.num_picked;
    }
    if (listed && num_entries <= kRanked) {
      // everything that is left fits one wave
      u64 *const units = lds.bins; // (nothing else is in the bins now)
      rank_entries(entries, num_entries, [&](int rank, u64 e) __attribute__((always_inline)) {
        units[rank] = units_of(entry_logit(e));
      });
      if (wave == 0) {
        const int n = num_entries < (int)k ? num_entries : (int)k;
        u64 w[kRankedEach], sum = 0;
#pragma unroll
        for (int i = 0; i < kRankedEach; ++i) {
          const int rank = lane * kRankedEach + i;
          w[i] = rank < n ? units[rank] : 0;
          sum += w[i];
        }
        const u64 upto = wave_scan_u64(sum);
        const u64 total = wave_sum_u64(sum);
        const u64 target = share_of(total);
        u64 run = upto - sum, kept_sum = 0;
        int kept = 0;
#pragma unroll
        for (int i = 0; i < kRankedEach; ++i) {
          const int rank = lane * kRankedEach + i;
          // (every filter keeps a front of the order)
          if (rank < n && (p_setting >= 1.0 || run < target) && entry_logit(lds.ranked[rank]) >= floor_x) {
            ++kept;
            kept_sum += w[i];
          }
          run += w[i];
        }
        kept_sum = wave_sum_u64(kept_sum);
        const int all_kept = (int)wave_sum_u64((u64)kept);
        if (lane == 0) lds.listed = all_kept, lds.found_value = kept_sum;
      }
      __syncthreads();
      // in index order: the threads of an entry sum the kept masses up to its index
      const int n = lds.listed, share = share_for(n), i = tid >> share, part = tid & ((1 << share) - 1);
      const u64 total = lds.found_value, target = drawn_of(total);
      u64 before = 0;
      if (i < n) {
        const int index = entry_index(lds.ranked[i]);
#pragma unroll 8
        for (int j = part; j < n; j += 1 << share) before += entry_index(lds.ranked[j]) < index ? units[j] : 0;
        if (share >= 1) before += dpp_u64<0xB1>(before);
        if (share == 2) before += dpp_u64<0x4E>(before);
      }
      if (wave == kWaves - 1) { // (hardly ever one of those that counted)
        const double log_total = log_of(total);
        if (lane == 0) lds.log_total = log_total;
      }
      __syncthreads();
      if (i < n && part == 0 && before <= target && before + units[i] > target)
        finish(entry_index(lds.ranked[i]), entry_logit(lds.ranked[i]), lds.log_total);
      return;
    }
    if (listed) {
      cut_at(entry_border([](float) __attribute__((always_inline)) -> u64 { return 1; }, k));
    } else { // every logit, where there are more than k of them to count
      clear_bins();
      u64 count = 0;
      all_again([&](float, int) __attribute__((always_inline)) { ++count; });
      count = wave_sum_u64(count);
      if (lane == 0) lds.bins[wave] = count;
      __syncthreads();
      const BinScan<kThreads> s = scan_bins<kThreads>(lds);
      __syncthreads();
      if (s.total > k) set_cut(by_bits(all_again, one_each, k), 1);
    }
  }

  // Top-p over what is left: the hint, then the exact pass. Logits above `sure_x` are
  // surely kept, those from `window_x` up to it are listed.
  float sure_x = -INFINITY, window_x = INFINITY;
  bool window = false;
  if (p_setting < 1.0) {
    // 2048 steps over 2^26 of mass; what is smaller is in the last one and counts as nothing
    constexpr float kPerHalving = (float)(kBins - 1) / 26.0f;
    const float per_step = (float)fmin(kPerHalving * per_unit, 1.0e30);
#pragma unroll
    for (int b = 0; b < kBinsEach; ++b) lds.counts[tid + b * kThreads] = 0;
    const uint32_t beside = kBins + lane; // (what the steps do not hold goes here, a place per lane)
    __syncthreads();
    for_chunks([&](int c, const V &v) __attribute__((always_inline)) {
      float x[kVec];
      uint32_t step[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) x[e] = static_cast<float>(v[e]);
      if (cutting)
#pragma unroll
        for (int e = 0; e < kVec; ++e) x[e] = in_front(x[e], first_of(c, at_lane) + e) ? x[e] : -INFINITY;
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        step[e] = (uint32_t)fminf((top - x[e]) * per_step, (float)(kBins + kWave));
        step[e] = step[e] < beside ? step[e] : beside;
      }
#pragma unroll
      for (int e = 0; e < kVec; ++e) atomicAdd(&lds.counts[step[e]], 1u);
    });
    __syncthreads();
    // (2^40 to the largest mass, each taken at the middle of its step)
    BinScan<kThreads> s;
#pragma unroll
    for (int i = 0; i < kBinsEach; ++i) {
      const int b = s.bin(i);
      s.v[i] = b == kBins - 1 ? 0 : (u64)((float)lds.counts[b] * __builtin_amdgcn_exp2f(40.0f - ((float)b + 0.5f) / kPerHalving));
    }
    s = scan_values(lds, s);
    // Every mass is off by at most a factor 1 +- 0.0044, so a share p by at most 0.0088 p (1 - p).
    const u64 target = share_of(s.total);
    const u64 slack = (u64)((double)s.total * (0.009 * p_setting * (1.0 - p_setting) + 1.0e-5));
    at_target(s, target > slack ? target - slack : 1,
              [&](int at, u64, u64) __attribute__((always_inline)) { lds.found_at = at; });
    at_target(s, target + slack < s.total ? target + slack : s.total,
              [&](int at, u64, u64) __attribute__((always_inline)) { lds.found_too = at; });
    __syncthreads();
    const int from = lds.found_at, to = lds.found_too;
    sure_x = from == 0 ? INFINITY : top - ((float)from - 0.25f) / per_step;
    window_x = top - ((float)to + 1.25f) / per_step;
    window = true;
  }
  // Where min-p cuts above the window, nothing in the window stays: the logits that
  // min-p keeps are the answer if top-p's share is not reached before the last of them.
  const bool by_floor = window && floor_x > sure_x;
  if (by_floor) window_x = INFINITY;
  if (by_floor || !window) sure_x = next_below(floor_x);
  auto kept_units = [&](float x, int i) __attribute__((always_inline)) -> u64 {
    return in_front(x, i) && x >= floor_x ? units_of(x) : 0;
  };
  auto kept_of = [&](const V &v, int first, u64 (&w)[kVec]) __attribute__((always_inline)) {
#pragma unroll
    for (int e0 = 0; e0 < kVec; e0 += 4) {
      float x[4];
      double m[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = static_cast<float>(v[e0 + e]);
      rounded_masses(x, m);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e0 + e] = in_front(x[e], first + e0 + e) && x[e] >= floor_x ? __builtin_bit_cast(u64, m[e]) & kMassBits : 0;
    }
  };
  while (true) {
    if (tid == 0) lds.num_picked = 0;
    start_list();
    clear_bins();
    // Whole numbers, at most 2^53 for a thread's logits: 64-bit floats hold their sums exactly.
    double all = 0.0, kept = 0.0; // what top-p is a share of, and what it surely keeps
    for_chunks([&](int c, const V &v) __attribute__((always_inline)) {
#pragma unroll
      for (int e0 = 0; e0 < kVec; e0 += 4) { // (four at a time: the masses of eight do not fit the registers)
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = static_cast<float>(v[e0 + e]);
        if (cutting)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = in_front(x[e], first_of(c, at_lane) + e0 + e) ? x[e] : -INFINITY;
        double w[4];
        rounded_masses(x, w);
        bool near = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] -= kRounding;
          all += w[e];
          // (the upper half alone says nothing: the lower one is then a number below 2^-1022)
          const u64 bits = __builtin_bit_cast(u64, w[e]);
          const uint32_t upper = x[e] > sure_x ? (uint32_t)(bits >> 32) : 0u;
          kept += __builtin_bit_cast(double, (u64)upper << 32 | (uint32_t)bits);
          near |= (x[e] >= window_x) & (x[e] <= sure_x);
        }
        if (near)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (x[e] >= window_x && x[e] <= sure_x && w[e] > 0.0) append(x[e], first_of(c, at_lane) + e0 + e);
          }
        __builtin_amdgcn_sched_barrier(0);
      }
    });
    const u64 wave_kept = wave_sum_u64((u64)kept), wave_all = wave_sum_u64((u64)all);
    if (lane == 0) lds.wave_kept[wave] = wave_kept, lds.wave_all[wave] = wave_all;
    __syncthreads();
    if (!window) break;
    const u64 total = wave_sum_u64(lane < kWaves ? lds.wave_all[lane] : 0);
    const u64 above = wave_sum_u64(lane < kWaves ? lds.wave_kept[lane] : 0);
    const u64 target = share_of(total);
    const int n = lds.listed;
    if (by_floor && above <= target) break;
    if (!by_floor && n <= kListed) {
      // the listed ones by their place between the window's ends, in the order of the logits
      const float from = fminf(sure_x, top), range = from - window_x;
      const float per_bin = range > 0.f ? fminf((float)(kBins - 1) / range, 1.0e30f) : 0.f;
      auto bin_of = [&](float x) __attribute__((always_inline)) {
        return (int)fminf((from - x) * per_bin, (float)(kBins - 1));
      };
      for_listed([&](float x, int) __attribute__((always_inline)) { atomicAdd(&lds.bins[bin_of(x)], units_of(x)); });
      __syncthreads();
      const BinScan<kThreads> s = scan_bins<kThreads>(lds);
      if (target > above && target <= above + s.total) {
        // the border is among the listed ones: in this bin
        const Found f = find_bin(lds, s, target - above);
        for_listed([&](float x, int i) __attribute__((always_inline)) {
          if (bin_of(x) == f.at) pick(x, i);
        });
        __syncthreads();
        const int picked = lds.num_picked;
        if (picked == 1) {
          cut_at(lds.picked[0]);
        } else if (picked <= kRanked) {
          rank_entries(lds.picked, picked, [](int, u64) __attribute__((always_inline)) {});
          if (wave == 0) { // each lane takes ranks one behind the other
            const int each = (picked + kWave - 1) / kWave, first = lane * each;
            const int last = first + each < picked ? first + each : picked;
            u64 sum = 0;
            for (int i = first; i < last; ++i) sum += units_of(entry_logit(lds.ranked[i]));
            u64 run = above + f.before + wave_scan_u64(sum) - sum;
            for (int i = first; i < last; ++i) {
              const u64 w = units_of(entry_logit(lds.ranked[i]));
              if (run < target && run + w >= target) lds.found_at = i; // exactly one
              run += w;
            }
          }
          __syncthreads();
          cut_at(lds.ranked[lds.found_at]);
        } else {
          cut_at(entry_border(units_of, target - above));
        }
        // those in front of it join the sums of their waves
        for_listed([&](float x, int i) __attribute__((always_inline)) {
          const u64 w = kept_units(x, i);
          if (w) atomicAdd(&lds.wave_kept[(i + lead) / kVec / kWave / chunks], w);
        });
        break;
      }
    }
    // the hint was off, or its step too full: the exact search, and the pass again without a window
    const Border b = by_bits(all_again, [&](float x, int i) __attribute__((always_inline)) -> u64 {
      return in_front(x, i) ? units_of(x) : 0;
    }, target);
    set_cut(b, units_of(key_value(b.key)));
    window = false;
    window_x = INFINITY;
    sure_x = next_below(floor_x);
  }
  __syncthreads();
  // The draw: the wave in whose run of the row the running mass passes the target, its
  // chunk (every wave sums some), and the logit in it.
  const u64 waves_upto = wave_scan_u64(lane < kWaves ? lds.wave_kept[lane] : 0);
  const u64 total = lane_u64(waves_upto, kWaves - 1);
  const u64 target = drawn_of(total);
  const int from = __popcll(__ballot(lane < kWaves && waves_upto <= target)); // (< kWaves: the target is below the total)
  u64 before = from > 0 ? lane_u64(waves_upto, from - 1) : 0;
  const int first_chunk = from * chunks;
  if (wave == kWaves - 1) { // (the wave that has the fewest of the chunks below)
    const double log_total = log_of(total);
    if (lane == 0) lds.log_total = log_total;
  }
  V v{};
  u64 w[kVec];
  auto weigh = [&](int c) __attribute__((always_inline)) {
    const int piece = (first_chunk + c) * kWave + lane;
    v = load(piece);
    kept_of(v, first_in(piece), w);
  };
  int weighed = -1; // the chunk that v and w are of
#pragma unroll 1
  for (int c = wave; c < chunks; c += kWaves) {
    weigh(c);
    u64 sum = 0;
#pragma unroll
    for (int e = 0; e < kVec; ++e) sum += w[e];
    sum = wave_sum_u64(sum);
    if (lane == 0) lds.list[c] = sum; // (the list is read no more)
    weighed = c;
  }
  __syncthreads();
  int c = 0;
#pragma unroll 1
  while (true) { // 64 chunks at a time: those that end before the target
    const u64 upto = before + wave_scan_u64(c + lane < chunks ? lds.list[c + lane] : 0);
    const int passed = __popcll(__ballot(c + lane < chunks - 1 && upto <= target));
    if (passed > 0) before = lane_u64(upto, passed - 1);
    c += passed;
    if (passed < kWave) break;
  }
  if (wave != c % kWaves) return;
  if (c != weighed) weigh(c);
  inside_chunk(v, w, (first_chunk + c) * kWave + lane, before, target, [&](int index, float x)
                   __attribute__((always_inline)) { finish(index, x, lds.log_total); });
}

// Logits a row may have: its chunks have to fit the bins, and the list.
constexpr int64_t kMaxVocab = 500000;
// A block of 1024 threads per row while every row gets a CU of its own; smaller blocks gain where two share a CU. In us,
// 512 threads against 1024, 50257 logits, top-p 0.92: 256 rows 46 against 37 in fp32, 39 against 34 in bf16; 257 rows 56
// against 62, 53 against 62; 512 rows 65 against 69, 58 against 67; 1000 rows 118 against 130, 106 against 130. (With top-k 50:
// 256 rows 23 against 18, 257 24 against 28, 768 50 against 50 in fp32; without filters 31, 25, 40, 42, 66, 69.)
constexpr int64_t kRowsAtOnce = 256;
static_assert(kMaxVocab + 8 <= (int64_t)kBins * kWave * 4 - kMostWaves * kWave * 4, "a bin per chunk");

template <typename T, int kThreads>
int launch_sample_threads(const SampleArgs &a, int64_t rows, hipStream_t stream) {
  constexpr int kChunk = kThreads * Io<T>::kVec, kMostInLds = most_in_lds(kThreads);
  const int chunks = (a.vocab + Io<T>::kVec - 1 + kChunk - 1) / kChunk;
  const int in_lds = chunks <= kInRegisters ? 0 : chunks - kInRegisters < kMostInLds ? chunks - kInRegisters : kMostInLds;
  const unsigned bytes = (unsigned)(sizeof(SampleLds) + (size_t)in_lds * kThreads * 16);
  constexpr unsigned kMostBytes = (unsigned)(sizeof(SampleLds) + (size_t)kMostInLds * kThreads * 16);
  static_assert(kMostBytes * (1024 / kThreads) <= 160 * 1024, "of a CU");
  const int s = raise_lds_limit(reinterpret_cast<const void *>(sample_kernel<T, kThreads>), kMostBytes, "oslo_sample");
  if (s != OSLO_OK) return s;
  sample_kernel<T, kThreads><<<dim3((unsigned)rows), dim3(kThreads), bytes, stream>>>(a);
  return check_launch("sample");
}

template <typename T>
int launch_sample(const SampleArgs &a, int64_t rows, hipStream_t stream) {
  if (rows > kRowsAtOnce) return launch_sample_threads<T, 512>(a, rows, stream);
  return launch_sample_threads<T, 1024>(a, rows, stream);
}

} // namespace
} // namespace oslo

extern "C" int oslo_sample(int64_t *tokens, float *logprobs, const void *logits, const float *uniforms,
                           const float *temperatures, double temperature, const int32_t *top_ks,
                           int64_t top_k, const float *top_ps, double top_p, const float *min_ps,
                           double min_p, int64_t rows, int64_t vocab, int64_t row_stride, int dtype,
                           oslo_stream_t stream) {
  using namespace oslo;
  if (rows < 0 || vocab < 0 || row_stride < 0) return fail(OSLO_E_BAD_ARG, "oslo_sample: negative size");
  if (dtype != OSLO_F32 && dtype != OSLO_F16 && dtype != OSLO_BF16) return fail(OSLO_E_BAD_ARG, "unknown dtype %d", dtype);
  if (!temperatures && !(temperature >= 0.0)) return fail(OSLO_E_BAD_ARG, "oslo_sample: the temperature must not be negative");
  if (!top_ks && top_k < 0) return fail(OSLO_E_BAD_ARG, "oslo_sample: top_k must not be negative");
  if (!top_ps && !(top_p >= 0.0)) return fail(OSLO_E_BAD_ARG, "oslo_sample: top_p must not be negative");
  if (!min_ps && !(min_p >= 0.0 && min_p <= 1.0)) return fail(OSLO_E_BAD_ARG, "oslo_sample: min_p must be in [0, 1]");
  if (rows == 0) return OSLO_OK;
  if (vocab == 0) return fail(OSLO_E_BAD_ARG, "oslo_sample: no logits to draw from");
  if (vocab > kMaxVocab) return fail(OSLO_E_UNSUPPORTED, "oslo_sample: more than %lld logits a row", (long long)kMaxVocab);
  if (rows > (int64_t)0x7fffffff) return fail(OSLO_E_UNSUPPORTED, "oslo_sample: too many rows for one launch");
  if (!tokens || !logits || !uniforms) return fail(OSLO_E_BAD_ARG, "oslo_sample: null pointer");
  SampleArgs a;
  a.tokens = tokens, a.logprobs = logprobs, a.logits = logits, a.row_stride = row_stride, a.uniforms = uniforms;
  // (Logits that differ do so by 2^-149 at least: from here down all but the largest have mass 0, and the reciprocal
  // would leave the range of 64 bits. Temperatures of a row's own have 32 bits and cannot come near.)
  constexpr double kLeastTemperature = 1.0e-300;
  a.temperature = {temperatures, temperature > 0.0 && temperature < kLeastTemperature ? kLeastTemperature : temperature};
  a.top_k = {top_ks, (double)top_k};
  a.top_p = {top_ps, top_p};
  a.min_p = {min_ps, min_p};
  a.vocab = (int)vocab;
  int log2_vocab = 0;
  while (((int64_t)1 << log2_vocab) < vocab) ++log2_vocab;
  a.mass_bits = 61 - log2_vocab < 49 ? 61 - log2_vocab : 49; // (a thread's sum is at most 2^53)
  hipStream_t st = static_cast<hipStream_t>(stream);
  OSLO_DISPATCH_DTYPE(dtype, return launch_sample<T>(a, rows, st));
  return OSLO_OK;
}
