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
// too: exp in 64 bits, times 2^S, rounded (S = 62 - ceil(log2 vocabulary), 46 at
// fifty thousand tokens; a rounding of 2^-47 of the largest mass, ten million
// times finer than a 32-bit sum). Sums of whole numbers are exact in any order:
// histograms may use atomics and every run gives the same token.
//
// One block of 1024 threads takes a row.
// Every filter is a selection "where does the running weight along the order
// reach a target": a histogram over 2048 steps of the distance to the largest
// logit finds the step, three more over the bits of the logits inside that step
// find the logit.

#include "common.hpp"

namespace oslo {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr int kBins = 2048;

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

// 2^y for y <= 0: y = n + f with |f| <= 1/2, 2^f = e^(f ln 2) by its Taylor series to the
// eleventh power (the next term is below 2^-46 of the result), times 2^n.
__device__ __forceinline__ double exp2_of(double y) {
  if (!(y > -1100.0)) return 0.0; // (below the smallest double)
  const double n = __builtin_rint(y);
  const double z = (y - n) * 0.69314718055994530942;
  double s = 1.0 / 39916800.0;
  s = __builtin_fma(s, z, 1.0 / 3628800.0);
  s = __builtin_fma(s, z, 1.0 / 362880.0);
  s = __builtin_fma(s, z, 1.0 / 40320.0);
  s = __builtin_fma(s, z, 1.0 / 5040.0);
  s = __builtin_fma(s, z, 1.0 / 720.0);
  s = __builtin_fma(s, z, 1.0 / 120.0);
  s = __builtin_fma(s, z, 1.0 / 24.0);
  s = __builtin_fma(s, z, 1.0 / 6.0);
  s = __builtin_fma(s, z, 0.5);
  s = __builtin_fma(s, z, 1.0);
  s = __builtin_fma(s, z, 1.0);
  return __builtin_ldexp(s, (int)n);
}

__device__ __forceinline__ u64 shfl_xor_u64(u64 v, int mask) {
  const uint32_t lo = __shfl_xor((uint32_t)v, mask, kWave), hi = __shfl_xor((uint32_t)(v >> 32), mask, kWave);
  return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 wave_sum_u64(u64 v) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) v += shfl_xor_u64(v, d);
  return v;
}
__device__ __forceinline__ u64 shfl_up_u64(u64 v, int d) {
  const uint32_t lo = __shfl_up((uint32_t)v, d, kWave), hi = __shfl_up((uint32_t)(v >> 32), d, kWave);
  return (u64)hi << 32 | lo;
}
// Sum over the lanes up to and including this one.
__device__ __forceinline__ u64 wave_scan_u64(u64 v, int lane) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const u64 w = shfl_up_u64(v, d);
    if (lane >= d) v += w;
  }
  return v;
}

struct SampleLds {
  u64 bins[kBins];
  u64 wave_sums[kWaves];
  float wave_max[kWaves], wave_min[kWaves];
  u64 found_before; // results of a search, written by the one thread that finds them
  int found_at;
  int found_index;
  double found_mass;
};

// In bins[0 .. count) (count a multiple of the block or below it): the first bin
// at which the running sum reaches `target`, and the sum before it. Every thread
// gets the answer; the sum of all bins must reach the target.
__device__ __forceinline__ void find_bin(SampleLds &lds, int count, u64 target, int &bin, u64 &before) {
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const int per = (count + kThreads - 1) / kThreads; // consecutive bins of a thread
  u64 mine = 0;
  for (int i = 0; i < per; ++i) {
    const int b = tid * per + i;
    if (b < count) mine += lds.bins[b];
  }
  const u64 upto = wave_scan_u64(mine, lane);
  if (lane == kWave - 1) lds.wave_sums[wave] = upto;
  __syncthreads();
  u64 run = upto - mine;
  for (int w = 0; w < wave; ++w) run += lds.wave_sums[w];
  if (run < target && run + mine >= target) { // exactly one thread
    for (int i = 0; i < per; ++i) {
      const int b = tid * per + i;
      const u64 v = lds.bins[b];
      if (run + v >= target) {
        lds.found_at = b;
        lds.found_before = run;
        break;
      }
      run += v;
    }
  }
  __syncthreads();
  bin = lds.found_at;
  before = lds.found_before;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(const SampleArgs a) {
  constexpr int kVec = Io<T>::kVec; // logits of a 16-byte load
  constexpr int kChunk = kThreads * kVec;
  using V = RawVec<T, kVec>;
  __shared__ SampleLds lds;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int64_t row = blockIdx.x;
  const int vocab = a.vocab;
  const T *const logits = static_cast<const T *>(a.logits) + row * a.row_stride;
  // Rows of an odd number of logits begin anywhere: loads are 16-byte aligned, and
  // the row begins `lead` logits into the first.
  const int lead = (int)((reinterpret_cast<uintptr_t>(logits) & 15u) / sizeof(T));
  const int chunks = (vocab + lead + kChunk - 1) / kChunk;
  // index of the first logit of this thread's vector of chunk c (may be negative)
  auto first_of = [&](int c) __attribute__((always_inline)) { return c * kChunk + tid * kVec - lead; };
  auto load = [&](int c) __attribute__((always_inline)) {
    V v;
    const int i0 = first_of(c);
    if (i0 >= 0 && i0 + kVec <= vocab) {
      v = *reinterpret_cast<const V *>(logits + i0);
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        v[e] = i0 + e >= 0 && i0 + e < vocab ? logits[i0 + e] : static_cast<T>(-INFINITY);
    }
    return v;
  };
  // f(chunk, vector) for every vector of the row
  auto for_chunks = [&](auto &&f) __attribute__((always_inline)) {
#pragma unroll 1
    for (int c = 0; c < chunks; ++c) f(c, load(c));
  };
  auto value = [](const V &v, int e) __attribute__((always_inline)) {
    const float x = static_cast<float>(v[e]);
    return x != x ? -INFINITY : x;
  };

  // the largest logit, and the smallest finite one
  float top = -INFINITY, low = INFINITY;
  for_chunks([&](int, const V &v) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      const float x = value(v, e);
      top = fmaxf(top, x);
      low = fminf(low, x == -INFINITY ? INFINITY : x);
    }
  });
  top = wave_allreduce(top, OpMax());
  low = -wave_allreduce(-low, OpMax());
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

  const double temperature = a.temperature.at(row);
  const bool greedy = !(temperature > 0.0); // the first of the largest
  const double per_unit = greedy ? 0.0 : 1.4426950408889634074 / temperature;
  // mass of a logit, relative to the largest one's, and as a whole number of 2^-S
  auto mass_of = [&](float x) __attribute__((always_inline)) -> double {
    if (x == top) return 1.0; // (also where both are infinite)
    return greedy ? 0.0 : exp2_of(((double)x - (double)top) * per_unit);
  };
  const double unit = __builtin_ldexp(1.0, a.mass_bits);
  auto units_of = [&](double mass) __attribute__((always_inline)) -> u64 {
    // (below 2^52: adding 2^52 leaves the rounded whole number in the low bits)
    const double shifted = __builtin_fma(mass, unit, 4503599627370496.0);
    return __builtin_bit_cast(u64, shifted) & 0xfffffffffffffull;
  };

  // Where, along the order, the running weight reaches `target`: the key of the
  // logit, and the weight that is missing there. `weight(x)` is the whole-number
  // weight of a logit, 0 for those not to be counted.
  const float span = top - low;
  const float per_step = span > 0.f && span < 3.0e38f ? (float)(kBins - 1) / span : 0.f;
  auto step_of = [&](float x) __attribute__((always_inline)) -> int { // falls as x rises
    return x == top ? 0 : (int)fminf((top - x) * per_step, (float)(kBins - 1));
  };
  auto select = [&](auto &&weight, u64 target, uint32_t &key, u64 &missing) __attribute__((always_inline)) {
    for (int b = tid; b < kBins; b += kThreads) lds.bins[b] = 0;
    __syncthreads();
    for_chunks([&](int, const V &v) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const float x = value(v, e);
        const u64 w = weight(x);
        if (w) atomicAdd(&lds.bins[step_of(x)], w);
      }
    });
    __syncthreads();
    int step;
    u64 before;
    find_bin(lds, kBins, target, step, before);
    target -= before;
    // inside the step: the bits of the key from the top, larger keys first
    uint32_t prefix = 0;
    int bits = 0;
#pragma unroll 1
    for (int level = 0; level < 3; ++level) {
      const int take = level == 2 ? 10 : 11, shift = 32 - bits - take;
      for (int b = tid; b < kBins; b += kThreads) lds.bins[b] = 0;
      __syncthreads();
      for_chunks([&](int, const V &v) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const float x = value(v, e);
          if (x == -INFINITY || step_of(x) != step) continue;
          const uint32_t k = order_key(x);
          if (bits && (k >> (32 - bits)) != prefix) continue;
          const u64 w = weight(x);
          if (w) atomicAdd(&lds.bins[((1u << take) - 1) - ((k >> shift) & ((1u << take) - 1))], w);
        }
      });
      __syncthreads();
      int bin;
      find_bin(lds, 1 << take, target, bin, before);
      target -= before;
      prefix = prefix << take | (((1u << take) - 1) - (uint32_t)bin);
      bits += take;
    }
    key = prefix;
    missing = target;
  };
  // Sum of a weight over the row.
  auto total_of = [&](auto &&weight) __attribute__((always_inline)) -> u64 {
    u64 sum = 0;
    for_chunks([&](int c, const V &v) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) sum += weight(value(v, e), first_of(c) + e);
    });
    sum = wave_sum_u64(sum);
    __syncthreads();
    if (lane == 0) lds.wave_sums[wave] = sum;
    __syncthreads();
    sum = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += lds.wave_sums[w];
    __syncthreads();
    return sum;
  };
  // The first index, in index order, at which the running weight exceeds `target`.
  auto index_past = [&](auto &&weight, u64 target, double &mass) __attribute__((always_inline)) -> int {
    u64 run = 0; // weight before the chunk
    int answer = -1;
    auto one = [&](int c, const V &v) __attribute__((always_inline)) {
      if (answer >= 0) return;
      u64 w[kVec], mine = 0;
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        w[e] = weight(value(v, e), first_of(c) + e);
        mine += w[e];
      }
      const u64 upto = wave_scan_u64(mine, lane);
      if (lane == kWave - 1) lds.wave_sums[wave] = upto;
      __syncthreads();
      u64 before = run, all = 0;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) {
        if (i < wave) before += lds.wave_sums[i];
        all += lds.wave_sums[i];
      }
      __syncthreads();
      if (run + all > target) { // in this chunk (the same for every thread)
        u64 at = before + upto - mine;
        if (at <= target && at + mine > target) { // exactly one thread
#pragma unroll
          for (int e = 0; e < kVec; ++e) {
            if (at <= target && at + w[e] > target) {
              lds.found_index = first_of(c) + e;
              lds.found_mass = (double)value(v, e);
            }
            at += w[e];
          }
        }
        __syncthreads();
        answer = lds.found_index;
        mass = lds.found_mass;
      }
      run += all;
    };
    for_chunks(one);
    return answer;
  };

  // the kept front of the order: logits with a key above `cut_key`, and those with
  // that key and an index up to `cut_index`
  uint32_t cut_key = 0;
  int cut_index = vocab;
  auto in_front = [&](float x, int index) __attribute__((always_inline)) {
    const uint32_t k = order_key(x);
    return x != -INFINITY && (k > cut_key || (k == cut_key && index <= cut_index));
  };
  auto set_cut = [&](uint32_t key, u64 ties) __attribute__((always_inline)) { // the first `ties` of the logits with this key
    cut_key = key;
    double unused;
    cut_index = index_past([&](float x, int) __attribute__((always_inline)) -> u64 { return order_key(x) == key ? 1 : 0; },
                           ties - 1, unused);
  };
  const double k_setting = a.top_k.at(row);
  if (greedy || (k_setting > 0.0 && k_setting < (double)vocab)) {
    const u64 k = greedy ? 1 : (u64)k_setting;
    // (with fewer finite logits than k there is nothing to cut)
    const u64 finite = total_of([&](float x, int) __attribute__((always_inline)) -> u64 { return x == -INFINITY ? 0 : 1; });
    if (finite > k) {
      uint32_t key;
      u64 ties;
      select([&](float x) __attribute__((always_inline)) -> u64 { return x == -INFINITY ? 0 : 1; }, k, key, ties);
      set_cut(key, ties);
    }
  }
  const double p_setting = greedy ? 1.0 : a.top_p.at(row);
  if (p_setting < 1.0) {
    const u64 all = total_of([&](float x, int i) __attribute__((always_inline)) -> u64 {
      return in_front(x, i) ? units_of(mass_of(x)) : 0;
    });
    const double wanted = __builtin_ceil((p_setting > 0.0 ? p_setting : 0.0) * (double)all);
    u64 target = wanted < 1.0 ? 1 : (u64)wanted;
    if (target > all) target = all;
    const uint32_t floor_key = cut_key;
    uint32_t key;
    u64 missing;
    select([&](float x) __attribute__((always_inline)) -> u64 {
      return x != -INFINITY && order_key(x) >= floor_key ? units_of(mass_of(x)) : 0;
    }, target, key, missing);
    const float cut = __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
    const u64 each = units_of(mass_of(cut));
    const u64 ties = (missing + each - 1) / each;
    set_cut(key, ties);
  }
  const double min_mass = greedy ? 0.0 : fmin(a.min_p.at(row), 1.0); // (the largest always stays)
  auto kept_units = [&](float x, int i) __attribute__((always_inline)) -> u64 {
    if (!in_front(x, i)) return 0;
    const double mass = mass_of(x);
    return mass >= min_mass ? units_of(mass) : 0;
  };
  const u64 all = total_of(kept_units);
  double u = (double)a.uniforms[row];
  u = u >= 0.0 ? (u < 1.0 ? u : 0.99999994039535522) : 0.0;
  u64 target = (u64)(u * (double)all);
  if (target >= all) target = all - 1;
  double logit = 0.0;
  int token = index_past(kept_units, target, logit);
  if (tid == 0) {
    a.tokens[row] = token;
    if (a.logprobs)
      a.logprobs[row] = (float)(((float)logit == top ? 0.0 : (logit - (double)top) * (greedy ? 0.0 : 1.0 / temperature)) -
                                log((double)all / unit));
  }
}

template <typename T>
int launch_sample(const SampleArgs &a, int64_t rows, hipStream_t stream) {
  sample_kernel<T><<<dim3((unsigned)rows), dim3(kThreads), 0, stream>>>(a);
  return check_launch("sample");
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
  if (vocab > (int64_t)1 << 24) return fail(OSLO_E_UNSUPPORTED, "oslo_sample: more than 2^24 logits a row");
  if (rows > (int64_t)0x7fffffff) return fail(OSLO_E_UNSUPPORTED, "oslo_sample: too many rows for one launch");
  if (!tokens || !logits || !uniforms) return fail(OSLO_E_BAD_ARG, "oslo_sample: null pointer");
  SampleArgs a;
  a.tokens = tokens, a.logprobs = logprobs, a.logits = logits, a.row_stride = row_stride, a.uniforms = uniforms;
  a.temperature = {temperatures, temperature};
  a.top_k = {top_ks, (double)top_k};
  a.top_p = {top_ps, top_p};
  a.min_p = {min_ps, min_p};
  a.vocab = (int)vocab;
  int log2_vocab = 0;
  while (((int64_t)1 << log2_vocab) < vocab) ++log2_vocab;
  a.mass_bits = 62 - log2_vocab < 51 ? 62 - log2_vocab : 51;
  hipStream_t st = static_cast<hipStream_t>(stream);
  OSLO_DISPATCH_DTYPE(dtype, return launch_sample<T>(a, rows, st));
  return OSLO_OK;
}
