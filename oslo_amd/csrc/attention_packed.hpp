// What the two entry points of the packed attention check before they launch.
#pragma once

#include "attention.hpp"

namespace oslo {
namespace {

constexpr int kPackedPositions = 128; // positions of a sequence an entry of the list of blocks stands for

// `strides`: (head, token) of each of the `count` tensors, in elements. OSLO_OK
// (also for a call with nothing to do), or the error.
inline int check_packed(const char *name, const void *const *tensors, const int64_t *strides, int count,
                        float scale, const int32_t *blocks, int64_t num_blocks, int64_t tokens, int64_t max_length,
                        int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t window, int dtype) {
  if (num_blocks < 0 || tokens < 0 || max_length < 0 || heads < 0 || kv_heads < 0 || head_dim < 0 || window < 0)
    return fail(OSLO_E_BAD_ARG, "%s: negative size", name);
  if (dtype != OSLO_F16 && dtype != OSLO_BF16) {
    if (dtype == OSLO_F32) return fail(OSLO_E_UNSUPPORTED, "%s: fp16 and bf16 are taken, not fp32", name);
    return fail(OSLO_E_BAD_ARG, "unknown dtype %d", dtype);
  }
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(OSLO_E_UNSUPPORTED, "%s: heads of %lld features (64, 128 or 256 are taken)", name,
                (long long)head_dim);
  if (!(scale > 0.0f)) return fail(OSLO_E_BAD_ARG, "%s: the scale must be positive", name);
  if (kv_heads == 0 ? heads != 0 : heads % kv_heads != 0)
    return fail(OSLO_E_BAD_ARG, "%s: %lld query heads do not share %lld key/value heads evenly", name,
                (long long)heads, (long long)kv_heads);
  if (num_blocks == 0 || heads == 0 || tokens == 0) return OSLO_OK;
  if (max_length == 0 || max_length > tokens)
    return fail(OSLO_E_BAD_ARG, "%s: a longest sequence of %lld among %lld tokens", name, (long long)max_length,
                (long long)tokens);
  if (!blocks || !strides) return fail(OSLO_E_BAD_ARG, "%s: null pointer", name);
  // (starts and lengths are 32-bit in the list; the grid has an entry per block and query head)
  if (tokens > (int64_t)0x7fffffff || heads > 65535 || num_blocks > (int64_t)0x7fffffff / heads)
    return fail(OSLO_E_UNSUPPORTED, "%s: too many tokens or blocks for one launch", name);
  for (int i = 0; i < count; ++i) {
    if (!tensors[i]) return fail(OSLO_E_BAD_ARG, "%s: null pointer", name);
    if (!aligned16(tensors[i])) return fail(OSLO_E_UNSUPPORTED, "%s: tensors must be 16-byte aligned", name);
    const int64_t sh = strides[2 * i], st = strides[2 * i + 1];
    if (sh < 0 || st < head_dim || sh % 8 || st % 8)
      return fail(OSLO_E_UNSUPPORTED,
                  "%s: strides must be multiples of 8 elements, the token stride at least head_dim", name);
    // byte offsets inside one sequence of a head are 32-bit
    if (st > (int64_t)0x7fffffff / 2 / (max_length + kPackedPositions))
      return fail(OSLO_E_UNSUPPORTED, "%s: a sequence of a head exceeds 2 GiB", name);
  }
  return OSLO_OK;
}

inline PackedArgs packed_args(const int32_t *blocks, int64_t tokens, int64_t max_length, int64_t heads,
                              int64_t kv_heads) {
  PackedArgs p;
  p.blocks = blocks;
  p.tokens = tokens;
  p.max_length = (int)max_length;
  p.kv_heads = (int)kv_heads;
  p.group = (int)(heads / kv_heads);
  return p;
}

} // namespace
} // namespace oslo
