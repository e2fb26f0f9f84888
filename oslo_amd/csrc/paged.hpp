// The paged key/value cache: where a position of a sequence lies, and the 8-bit
// storage of its vectors.
//
// Pages [num_pages, kv_heads, page_size, head_dim]: the slots of one head of a
// page are consecutive rows. A table [sequences, max_pages] of page numbers says
// which page holds the positions [i * page_size, (i + 1) * page_size) of a
// sequence. Offsets into the pages are 64-bit.
//
// 8-bit storage: OCP e4m3 with one scale per (slot, head), a power of two 2^e
// kept as the byte e + 127 in [num_pages, kv_heads, page_size]. e is the least
// integer with max|x| <= 448 * 2^e (448 is e4m3's largest number). A power of two
// costs a floating-point format no precision (only the exponents move) and makes
// both directions exact but for the one rounding to e4m3: x * 2^-e and q * 2^e are
// exact in fp32, and q * 2^e is a bf16 or fp16 number wherever it is in the type's
// normal range, so the matrix cores read the values themselves, not roundings of
// them. In fp16 products below 2^-14 may be rounded, to multiples of 2^-24; those above 65504,
// which only a cache written in bf16 can hold, are infinite.
#pragma once

#include "common.hpp"

namespace oslo {

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));

struct PageMap {
  const int *table; // [sequences][max_pages]
  int sequences, max_pages, num_pages, kv_heads, page_shift;
};

// Exponent of the scale of a vector whose largest finite magnitude has the fp32
// bits `amax` (0: nothing but zeros, scale 1). Exponents below -126 are not
// needed by any 16-bit type's range; -126 keeps the byte above 0 and the factor
// 2^-e finite.
__device__ __forceinline__ int scale_exponent(uint32_t amax) {
  if (amax == 0) return 0;
  const int e = (int)(amax >> 23) - 127 - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < -126 ? -126 : e;
}
__device__ __forceinline__ float exponent_to_scale(int biased) { // 2^(biased - 127), biased in 1 .. 254
  return __builtin_bit_cast(float, (uint32_t)biased << 23);
}

// Two e4m3 numbers (the low or the high half of a word) times 2^e, as T (exact in the
// type's normal range).
template <typename T>
using Pair = typename VecOf<T, 2>::type;
template <bool HIGH>
__device__ __forceinline__ Pair<bf16> e4m3_pair(uint32_t word, float scale, bf16) {
  return __builtin_bit_cast(Pair<bf16>, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, HIGH));
}
template <bool HIGH>
__device__ __forceinline__ Pair<f16> e4m3_pair(uint32_t word, float scale, f16) {
  return __builtin_bit_cast(Pair<f16>, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, scale, HIGH));
}

} // namespace oslo

namespace oslo {

// What every entry point over the pages checks; fills the map. Page sizes are
// powers of two from 16 (a tile of 16 keys of the attention lies in one page) to 4096.
inline int check_pages(const char *name, const void *key_pages, const void *value_pages, const void *key_scales,
                       const void *value_scales, const int32_t *table, int64_t sequences, int64_t max_pages,
                       int64_t num_pages, int64_t kv_heads, int64_t page_size, int64_t head_dim, int dtype,
                       PageMap *map) {
  if (sequences < 0 || max_pages < 0 || num_pages < 0 || kv_heads < 0 || page_size < 0 || head_dim < 0)
    return fail(OSLO_E_BAD_ARG, "%s: negative size", name);
  if (dtype != OSLO_F16 && dtype != OSLO_BF16) {
    if (dtype == OSLO_F32) return fail(OSLO_E_UNSUPPORTED, "%s: fp16 and bf16 are taken, not fp32", name);
    return fail(OSLO_E_BAD_ARG, "unknown dtype %d", dtype);
  }
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(OSLO_E_UNSUPPORTED, "%s: heads of %lld features (64, 128 or 256 are taken)", name,
                (long long)head_dim);
  int shift = 4;
  while (shift < 12 && ((int64_t)1 << shift) < page_size) ++shift;
  if (((int64_t)1 << shift) != page_size)
    return fail(OSLO_E_UNSUPPORTED, "%s: pages of %lld positions (a power of two from 16 to 4096 is taken)", name,
                (long long)page_size);
  if ((key_scales == nullptr) != (value_scales == nullptr))
    return fail(OSLO_E_BAD_ARG, "%s: scales of keys and of values go together", name);
  if (kv_heads > 65535 || num_pages > (int64_t)0x7fffffff || sequences > (int64_t)0x7fffffff ||
      max_pages > ((int64_t)1 << 29 >> shift))
    return fail(OSLO_E_UNSUPPORTED, "%s: too many pages, sequences or heads", name);
  if (sequences > 0 && max_pages > 0 && kv_heads > 0 && num_pages > 0) {
    if (!key_pages || !value_pages || !table) return fail(OSLO_E_BAD_ARG, "%s: null pointer", name);
    if (!aligned16(key_pages) || !aligned16(value_pages) || !aligned16(key_scales) || !aligned16(value_scales))
      return fail(OSLO_E_UNSUPPORTED, "%s: pages and scales must be 16-byte aligned", name);
  }
  map->table = table;
  map->sequences = (int)sequences, map->max_pages = (int)max_pages, map->num_pages = (int)num_pages;
  map->kv_heads = (int)kv_heads, map->page_shift = shift;
  return OSLO_OK;
}

} // namespace oslo
