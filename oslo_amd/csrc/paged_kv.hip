// Keys and values of new tokens into the paged cache, and back out of it: one
// pass over the tokens' vectors each way, in 16 bits (a copy) or 8 bits
// (e4m3 with a power-of-two scale per token and head, paged.hpp):
//   write: e = least integer with max|x| <= 448 * 2^e;  q = round_to_e4m3(x * 2^-e), x in fp16
//          at most 61440 so that it can be read back
//   read:  x = q * 2^e
// The vector of one token and head is held by D / 8 lanes, 16 bytes each, so
// its largest magnitude is a reduction inside those lanes and it is read once.
// Bound by HBM.

#include <type_traits>

#include "paged.hpp"

namespace oslo {
namespace {

struct PagedKVArgs {
  void *key_pages, *value_pages;
  unsigned char *key_scales, *value_scales; // null: pages of T
  void *key, *value;                        // [tokens, kv_heads, D]; written by the read
  int64_t key_head, key_token, value_head, value_token; // element strides
  const int *rows, *positions;              // [tokens]: sequence and position of each token
  PageMap map;
  int64_t tokens;
};

// Slot (row of the pages) of token t's head, or -1 if the token has none: a
// sequence outside the table, a position outside the sequence's pages (negative
// ones mark tokens to pass over) or a page number outside the pool.
__device__ __forceinline__ int64_t slot_of(const PagedKVArgs &a, int64_t t, int head) {
  const int row = a.rows[t], position = a.positions[t];
  if (row < 0 || row >= a.map.sequences || position < 0) return -1;
  const int index = position >> a.map.page_shift;
  if (index >= a.map.max_pages) return -1;
  const int page = a.map.table[(int64_t)row * a.map.max_pages + index];
  if (page < 0 || page >= a.map.num_pages) return -1;
  const int slot = position & ((1 << a.map.page_shift) - 1);
  return ((((int64_t)page * a.map.kv_heads + head) << a.map.page_shift) + slot);
}

// Largest of the LANES values of an aligned group of lanes (8, 16 or 32).
template <int LANES>
__device__ __forceinline__ float max_over_lanes(float v) {
  v = fmaxf(v, dpp_move<0xB1>(v));
  v = fmaxf(v, dpp_move<0x4E>(v));
  v = fmaxf(v, dpp_move<0x141>(v));
  if constexpr (LANES >= 16) v = fmaxf(v, dpp_move<0x140>(v));
  if constexpr (LANES >= 32)
    v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, v), 0x401F)));
  return v;
}

// The largest number of the 8-bit storage that fp16 has: 240 * 2^8 (the next, 256 * 2^8, is
// infinity there). Larger ones of an fp16 vector, up to 65504, are taken to it: 6.2 % off, where
// the rounding to e4m3 may be off by 2^-4. Vectors with smaller scales hold nothing so large.
constexpr float kMostF16 = 61440.0f;

template <typename T, int D>
__device__ __forceinline__ void store_e4m3(unsigned char *pages, unsigned char *scales, int64_t slot, int part,
                                           const RawVec<T, 8> &raw) {
  float x[8];
  raw_to_f32<T, 8>(x, raw);
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, __builtin_isfinite(x[i]) ? fabsf(x[i]) : 0.f);
  amax = max_over_lanes<D / 8>(amax);
  const int e = scale_exponent(__builtin_bit_cast(uint32_t, amax));
  const float inverse = exponent_to_scale(127 - e);
  // (infinities and NaN have no scaled value: they are kept as NaN)
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float y = x[i];
    if constexpr (std::is_same<T, f16>::value) y = __builtin_amdgcn_fmed3f(y, -kMostF16, kMostF16);
    x[i] = __builtin_isfinite(x[i]) ? y * inverse : __builtin_nanf("");
  }
  u32x2 w;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j], x[4 * j + 1], 0, false);
    v = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j + 2], x[4 * j + 3], v, true);
    w[j] = (uint32_t)v;
  }
  if (slot >= 0) {
    __builtin_nontemporal_store(w, reinterpret_cast<u32x2 *>(pages + slot * D + 8 * part));
    if (part == 0) scales[slot] = (unsigned char)(e + 127);
  }
}

// A group of D / 8 lanes takes ROWS (token, head) rows, all loads of a thread issued
// before any is used; ROWS is 2 where the rows fill the card four times over, else 1
// (a decoding step: more, shorter blocks). One row against two, us, 8-bit: 256 tokens x 16 heads x 256 features
// 3.5, 4.4; 2048 tokens 12.8, 11.7; 4096 (where two begins) 23.1, 21.8; 17206 89, 80 (5.3 TB/s; 4 and 8 rows
// were slower than 2). 12 heads of 64: 256 tokens 3.2, 4.0; 17206 19.8, 20.1. In 16 bits two gain in the
// middle, 2048 tokens x 16 x 256 12.3, 10.6, and cost some at the end, 17206 tokens 86, 91.
template <typename T, int D, bool E4M3, int ROWS>
__global__ __launch_bounds__(kBlockThreads) void paged_kv_write_kernel(const PagedKVArgs a) {
  constexpr int kLanes = D / 8;
  constexpr int kRows = kBlockThreads / kLanes; // rows of a block at a time
  const int part = threadIdx.x % kLanes;
  const uint32_t row0 = blockIdx.x * (uint32_t)(kRows * ROWS) + threadIdx.x / kLanes;
  const uint32_t rows = (uint32_t)(a.tokens * a.map.kv_heads), heads = (uint32_t)a.map.kv_heads; // (below 2^31)
  using V = RawVec<T, 8>;
  V k[ROWS], v[ROWS];
  int64_t slot[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    uint32_t row = row0 + i * kRows;
    const bool live = row < rows;
    if (!live) row = rows - 1; // (the lanes of a group stay together)
    const int64_t t = row / heads;
    const int head = (int)(row % heads);
    k[i] = __builtin_nontemporal_load(
        reinterpret_cast<const V *>(static_cast<const T *>(a.key) + t * a.key_token + head * a.key_head + 8 * part));
    v[i] = __builtin_nontemporal_load(
        reinterpret_cast<const V *>(static_cast<const T *>(a.value) + t * a.value_token + head * a.value_head + 8 * part));
    slot[i] = live ? slot_of(a, t, head) : -1;
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    if constexpr (E4M3) {
      store_e4m3<T, D>(static_cast<unsigned char *>(a.key_pages), a.key_scales, slot[i], part, k[i]);
      store_e4m3<T, D>(static_cast<unsigned char *>(a.value_pages), a.value_scales, slot[i], part, v[i]);
    } else if (slot[i] >= 0) {
      __builtin_nontemporal_store(k[i], reinterpret_cast<V *>(static_cast<T *>(a.key_pages) + slot[i] * D + 8 * part));
      __builtin_nontemporal_store(v[i], reinterpret_cast<V *>(static_cast<T *>(a.value_pages) + slot[i] * D + 8 * part));
    }
  }
}

// One row per group of lanes: 77, 80, 85 and 97 us with 1, 2, 4 and 8 for 17206 tokens x 16 x 256, 8-bit
// (5.5 TB/s with 1).
template <typename T, int D, bool E4M3>
__global__ __launch_bounds__(kBlockThreads) void paged_kv_read_kernel(const PagedKVArgs a) {
  constexpr int kLanes = D / 8;
  constexpr int kRows = kBlockThreads / kLanes;
  const int part = threadIdx.x % kLanes;
  const uint32_t row = blockIdx.x * (uint32_t)kRows + threadIdx.x / kLanes;
  const uint32_t rows = (uint32_t)(a.tokens * a.map.kv_heads), heads = (uint32_t)a.map.kv_heads; // (below 2^31)
  if (row >= rows) return;
  using V = RawVec<T, 8>;
  using Raw = typename std::conditional<E4M3, u32x2, V>::type;
  Raw raw[2] = {Raw{}, Raw{}}; // (a token without a slot reads as zeros)
  int scale[2] = {127, 127};
  const int64_t slot = slot_of(a, row / heads, (int)(row % heads));
  if (slot >= 0) {
    constexpr int kElem = E4M3 ? 1 : (int)sizeof(T);
    const int64_t at = (slot * D + 8 * part) * kElem;
    raw[0] = __builtin_nontemporal_load(reinterpret_cast<const Raw *>(static_cast<const char *>(a.key_pages) + at));
    raw[1] = __builtin_nontemporal_load(reinterpret_cast<const Raw *>(static_cast<const char *>(a.value_pages) + at));
    if constexpr (E4M3) scale[0] = a.key_scales[slot], scale[1] = a.value_scales[slot];
  }
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    V x;
    if constexpr (E4M3) {
      const float factor = exponent_to_scale(scale[which]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const Pair<T> lo = e4m3_pair<false>(raw[which][j], factor, T()), hi = e4m3_pair<true>(raw[which][j], factor, T());
        x[4 * j] = lo[0], x[4 * j + 1] = lo[1], x[4 * j + 2] = hi[0], x[4 * j + 3] = hi[1];
      }
    } else {
      x = raw[which];
    }
    __builtin_nontemporal_store(x, reinterpret_cast<V *>(static_cast<T *>(which ? a.value : a.key) + (int64_t)row * D + 8 * part)); // (dense)
  }
}

template <typename T, int D, bool WRITE>
int launch_paged_kv(const PagedKVArgs &a, hipStream_t stream) {
  constexpr int kRows = kBlockThreads / (D / 8);
  const int64_t rows = a.tokens * a.map.kv_heads;
  auto grid = [&](int64_t per_block) { return dim3((unsigned)((rows + per_block - 1) / per_block)); };
  if constexpr (WRITE) {
    if (rows >= 4 * 256 * 8 * kRows) { // four times the blocks the card holds
      auto *kernel = a.key_scales ? paged_kv_write_kernel<T, D, true, 2> : paged_kv_write_kernel<T, D, false, 2>;
      kernel<<<grid(2 * kRows), dim3(kBlockThreads), 0, stream>>>(a);
    } else {
      auto *kernel = a.key_scales ? paged_kv_write_kernel<T, D, true, 1> : paged_kv_write_kernel<T, D, false, 1>;
      kernel<<<grid(kRows), dim3(kBlockThreads), 0, stream>>>(a);
    }
  } else {
    auto *kernel = a.key_scales ? paged_kv_read_kernel<T, D, true> : paged_kv_read_kernel<T, D, false>;
    kernel<<<grid(kRows), dim3(kBlockThreads), 0, stream>>>(a);
  }
  return check_launch(WRITE ? "paged_kv_write" : "paged_kv_read");
}

template <typename T, bool WRITE>
int launch_paged_kv_dim(const PagedKVArgs &a, int64_t head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 64: return launch_paged_kv<T, 64, WRITE>(a, stream);
    case 128: return launch_paged_kv<T, 128, WRITE>(a, stream);
    default: return launch_paged_kv<T, 256, WRITE>(a, stream);
  }
}

template <bool WRITE>
int paged_kv(const char *name, PagedKVArgs a, int64_t sequences, int64_t max_pages, int64_t num_pages,
             int64_t kv_heads, int64_t page_size, int64_t head_dim, int dtype, hipStream_t stream) {
  if (a.tokens < 0) return fail(OSLO_E_BAD_ARG, "%s: negative size", name);
  const int s = check_pages(name, a.key_pages, a.value_pages, a.key_scales, a.value_scales, a.map.table, sequences,
                            max_pages, num_pages, kv_heads, page_size, head_dim, dtype, &a.map);
  if (s != OSLO_OK) return s;
  if (a.tokens == 0 || kv_heads == 0) return OSLO_OK;
  if (!a.key || !a.value || !a.rows || !a.positions) return fail(OSLO_E_BAD_ARG, "%s: null pointer", name);
  if (!aligned16(a.key) || !aligned16(a.value))
    return fail(OSLO_E_UNSUPPORTED, "%s: key and value must be 16-byte aligned", name);
  if (a.key_head < 0 || a.key_token < 0 || a.value_head < 0 || a.value_token < 0 || a.key_head % 8 ||
      a.key_token % 8 || a.value_head % 8 || a.value_token % 8)
    return fail(OSLO_E_UNSUPPORTED, "%s: strides must be multiples of 8 elements", name);
  if (a.tokens > (int64_t)0x7fffffff / kv_heads)
    return fail(OSLO_E_UNSUPPORTED, "%s: too many tokens for one launch", name);
  if (dtype == OSLO_F16) return launch_paged_kv_dim<f16, WRITE>(a, head_dim, stream);
  return launch_paged_kv_dim<bf16, WRITE>(a, head_dim, stream);
}

} // namespace
} // namespace oslo

extern "C" int oslo_paged_kv_write(void *key_pages, void *value_pages, uint8_t *key_scales,
                                   uint8_t *value_scales, const void *key, const void *value,
                                   const int32_t *sequence, const int32_t *position,
                                   const int32_t *table, int64_t tokens, int64_t sequences,
                                   int64_t max_pages, int64_t num_pages, int64_t kv_heads,
                                   int64_t page_size, int64_t head_dim, const int64_t *strides,
                                   int dtype, oslo_stream_t stream) {
  using namespace oslo;
  if (!strides && tokens > 0) return fail(OSLO_E_BAD_ARG, "oslo_paged_kv_write: null pointer");
  PagedKVArgs a{};
  a.key_pages = key_pages, a.value_pages = value_pages, a.key_scales = key_scales, a.value_scales = value_scales;
  a.key = const_cast<void *>(key), a.value = const_cast<void *>(value);
  if (strides) a.key_head = strides[0], a.key_token = strides[1], a.value_head = strides[2], a.value_token = strides[3];
  a.rows = sequence, a.positions = position, a.map.table = table, a.tokens = tokens;
  return paged_kv<true>("oslo_paged_kv_write", a, sequences, max_pages, num_pages, kv_heads, page_size, head_dim,
                        dtype, static_cast<hipStream_t>(stream));
}

extern "C" int oslo_paged_kv_read(void *key, void *value, const void *key_pages,
                                  const void *value_pages, const uint8_t *key_scales,
                                  const uint8_t *value_scales, const int32_t *sequence,
                                  const int32_t *position, const int32_t *table, int64_t tokens,
                                  int64_t sequences, int64_t max_pages, int64_t num_pages,
                                  int64_t kv_heads, int64_t page_size, int64_t head_dim, int dtype,
                                  oslo_stream_t stream) {
  using namespace oslo;
  PagedKVArgs a{};
  a.key_pages = const_cast<void *>(key_pages), a.value_pages = const_cast<void *>(value_pages);
  a.key_scales = const_cast<uint8_t *>(key_scales), a.value_scales = const_cast<uint8_t *>(value_scales);
  a.key = key, a.value = value;
  a.rows = sequence, a.positions = position, a.map.table = table, a.tokens = tokens;
  return paged_kv<false>("oslo_paged_kv_read", a, sequences, max_pages, num_pages, kv_heads, page_size, head_dim,
                         dtype, static_cast<hipStream_t>(stream));
}
