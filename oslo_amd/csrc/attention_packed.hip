// Causal attention over sequences of different lengths laid one behind the
// other along one row of tokens (a batch of prompts, or documents packed into a
// training row), several query heads to a key/value head:
//   out[h, q, :] = sum over keys k <= q of q's own sequence of
//                  softmax_k(scale * Q[h, q, :] . K[h / group, k, :]) * V[h / group, k, :]
// The kernel is the prompt attention's (attention_prefill.hpp): a block takes
// 128 queries of one head of one sequence and streams that sequence's keys and
// values; no padding is computed and no position sees another sequence. What
// differs is where a block finds its work: a list of (start, length, block)
// entries, the ones with most keys first, instead of a regular grid.
//
// Bound by the matrix cores where sequences are long: 9 prompts of 8299 tokens, 16 heads of 256
// in bf16, 126 us for 84 Gflop, 0.67 Pflop/s. Short sequences cost that rate, in the dense kernel as here: 8 of 1024
// tokens 0.66 (dense 0.665), 4 of 2048 0.87 (0.83), 8 of 2048 0.815 (0.80), 1 of 8192 1.10 (1.10). 9144 tokens in
// 7 documents, 32 query heads on 8 of 128, 210 us with the statistics for the backward, 0.85 Pflop/s.
// With a window of 256 (8794 tokens, 20 heads of 128, fp16: 73 us) the blocks walk 12 tiles of 32 keys each
// and reading their queries and writing their outputs weighs as much as the products.
// For the backward the forward also writes what the output's rounding left out, 16 bits a
// feature more (7 us of the 73).

#include "attention_packed.hpp"
#include "attention_prefill.hpp"

namespace oslo {
namespace {

static_assert(kQueriesPerBlock == kPackedPositions, "an entry of the list is a block of the kernel");

template <typename T, int D>
int launch_packed(const PrefillArgs &a, int64_t num_blocks, hipStream_t stream) {
  constexpr unsigned kDynamic = prefill_lds_bytes<T, D>();
  auto *kernel = a.window > 0 ? attention_prefill_kernel<T, D, false, true, false, true>
                              : attention_prefill_kernel<T, D, false, false, false, true>;
  if (kDynamic > 64u * 1024u) {
    const int s = raise_lds_limit(reinterpret_cast<const void *>(kernel), kDynamic, "oslo_attention_packed_fwd");
    if (s != OSLO_OK) return s;
  }
  kernel<<<dim3((unsigned)(num_blocks * a.heads)), dim3(kBlockThreads), kDynamic, stream>>>(a);
  return check_launch("attention_packed_fwd");
}

template <typename T>
int launch_packed_dim(const PrefillArgs &a, int64_t num_blocks, int64_t head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 64: return launch_packed<T, 64>(a, num_blocks, stream);
    case 128: return launch_packed<T, 128>(a, num_blocks, stream);
    default: return launch_packed<T, 256>(a, num_blocks, stream);
  }
}

} // namespace
} // namespace oslo

extern "C" int oslo_attention_packed_fwd(void *out, void *out_low, float *lse, const void *q, const void *k,
                                         const void *v, const int32_t *blocks,
                                         int64_t num_blocks, float scale, int64_t tokens,
                                         int64_t max_length, int64_t heads,
                                         int64_t kv_heads, int64_t head_dim,
                                         int64_t window, const int64_t *strides,
                                         int dtype, oslo_stream_t stream) {
  using namespace oslo;
  const void *tensors[4] = {q, k, v, out};
  const int s = check_packed("oslo_attention_packed_fwd", tensors, strides, 4, scale, blocks, num_blocks, tokens,
                             max_length, heads, kv_heads, head_dim, window, dtype);
  if (s != OSLO_OK) return s;
  if (num_blocks == 0 || heads == 0 || tokens == 0) return OSLO_OK;
  PrefillArgs a{};
  if (!aligned16(out_low) || !aligned16(lse))
    return fail(OSLO_E_UNSUPPORTED, "oslo_attention_packed_fwd: lse and out_low must be 16-byte aligned");
  a.out = out, a.out_low = out_low, a.q = q, a.k = k, a.v = v, a.lse = lse;
  a.q_h = strides[0], a.q_s = strides[1];
  a.k_h = strides[2], a.k_s = strides[3];
  a.v_h = strides[4], a.v_s = strides[5];
  a.o_h = strides[6], a.o_s = strides[7];
  a.scale = scale;
  a.scale_log2e = scale * kLog2e;
  a.heads = (int)heads;
  a.window = window >= max_length ? 0 : (int)window;
  a.packed = packed_args(blocks, tokens, max_length, heads, kv_heads);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == OSLO_F16) return launch_packed_dim<f16>(a, num_blocks, head_dim, st);
  return launch_packed_dim<bf16>(a, num_blocks, head_dim, st);
}
