// Launches of the one-kernel prompt attention over [batch, head, position]
// tensors (the kernel: attention_prefill.hpp) and its entry points.

#include "attention_prefill.hpp"

namespace oslo {
namespace {

template <typename T, int D>
int launch_prefill_dim(const PrefillArgs &a, hipStream_t stream) {
  const dim3 grid((unsigned)(8 * a.head_groups * a.query_blocks));
  // All LDS of the kernel is dynamic. At head_dim 256 it exceeds the 64 KiB a
  // kernel gets unasked, so the limit is raised for the kernel (on the current
  // device; a host-side setting, not a stream operation), once.
  constexpr unsigned kDynamic = prefill_lds_bytes<T, D>();
  auto go = [&]<bool HAS_PAD, bool HAS_WINDOW>() -> int {
    auto *kernel = a.drop.drop ? attention_prefill_kernel<T, D, HAS_PAD, HAS_WINDOW, true>
                               : attention_prefill_kernel<T, D, HAS_PAD, HAS_WINDOW, false>;
    if (kDynamic > 64u * 1024u) {
      const int s = raise_lds_limit(reinterpret_cast<const void *>(kernel), kDynamic, "oslo_attention_prefill_fwd");
      if (s != OSLO_OK) return s;
    }
    kernel<<<grid, dim3(kBlockThreads), kDynamic, stream>>>(a);
    return check_launch("attention_prefill_fwd");
  };
  if (a.window > 0) {
    if (a.pad != nullptr) return go.template operator()<true, true>();
    return go.template operator()<false, true>();
  }
  if (a.pad != nullptr) return go.template operator()<true, false>();
  return go.template operator()<false, false>();
}

template <typename T>
int launch_prefill(const PrefillArgs &a, int head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 64: return launch_prefill_dim<T, 64>(a, stream);
    case 128: return launch_prefill_dim<T, 128>(a, stream);
    default: return launch_prefill_dim<T, 256>(a, stream);
  }
}

} // namespace
} // namespace oslo

namespace {
int prefill_entry(void *out, float *lse, const oslo::DropArgs &drop, const void *q,
                  const void *k, const void *v,
                  const float *pad, float scale, int64_t batch, int64_t heads,
                  int64_t S, int64_t head_dim, int64_t window,
                  const int64_t *strides, int dtype, oslo_stream_t stream) {
  using namespace oslo;
  if (batch < 0 || heads < 0 || S < 0 || head_dim < 0 || window < 0)
    return fail(OSLO_E_BAD_ARG, "oslo_attention_prefill_fwd: negative size");
  if (dtype != OSLO_F16 && dtype != OSLO_BF16) {
    if (dtype == OSLO_F32)
      return fail(OSLO_E_UNSUPPORTED, "oslo_attention_prefill_fwd: fp16 and bf16 are taken, not fp32");
    return fail(OSLO_E_BAD_ARG, "unknown dtype %d", dtype);
  }
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(OSLO_E_UNSUPPORTED,
                "oslo_attention_prefill_fwd: heads of %lld features (64, 128 or 256 are taken)",
                (long long)head_dim);
  if (!(scale > 0.0f))
    return fail(OSLO_E_BAD_ARG, "oslo_attention_prefill_fwd: the scale must be positive");
  if (batch == 0 || heads == 0 || S == 0) return OSLO_OK;
  if (!out || !q || !k || !v || !strides)
    return fail(OSLO_E_BAD_ARG, "oslo_attention_prefill_fwd: null pointer");
  if (batch * heads > (int64_t)0x7fffffff / 8)
    return fail(OSLO_E_UNSUPPORTED, "oslo_attention_prefill_fwd: too many heads for one launch");
  const void *ptrs[4] = {q, k, v, out};
  for (int i = 0; i < 4; ++i) {
    if (!aligned16(ptrs[i]))
      return fail(OSLO_E_UNSUPPORTED, "oslo_attention_prefill_fwd: tensors must be 16-byte aligned");
    const int64_t sb = strides[3 * i], sh = strides[3 * i + 1], ss = strides[3 * i + 2];
    if (sb < 0 || sh < 0 || ss < head_dim || sb % 8 || sh % 8 || ss % 8)
      return fail(OSLO_E_UNSUPPORTED,
                  "oslo_attention_prefill_fwd: strides must be multiples of 8 elements, "
                  "the position stride at least head_dim");
    // byte offsets inside one (batch, head) slice are 32-bit
    if ((S + kQueriesPerBlock) * ss * 2 > (int64_t)0x7fffffff)
      return fail(OSLO_E_UNSUPPORTED, "oslo_attention_prefill_fwd: a head's slice exceeds 2 GiB");
  }
  if (pad != nullptr && (S % 4 != 0 || !aligned16(pad)))
    return fail(OSLO_E_UNSUPPORTED,
                "oslo_attention_prefill_fwd: with a padding mask S must be a multiple of 4 and the mask 16-byte aligned");
  PrefillArgs a;
  if (drop.drop && S % 8 != 0)
    return fail(OSLO_E_UNSUPPORTED,
                "oslo_attention_prefill_fwd_lse: with attention dropout S must be a multiple of 8");
  a.out = out, a.q = q, a.k = k, a.v = v, a.pad = pad, a.lse = lse, a.drop = drop;
  a.q_b = strides[0], a.q_h = strides[1], a.q_s = strides[2];
  a.k_b = strides[3], a.k_h = strides[4], a.k_s = strides[5];
  a.v_b = strides[6], a.v_h = strides[7], a.v_s = strides[8];
  a.o_b = strides[9], a.o_h = strides[10], a.o_s = strides[11];
  a.scale = scale;
  a.scale_log2e = scale * kLog2e;
  a.S = (int)S;
  a.heads = (int)heads;
  a.batch_heads = (int)(batch * heads);
  a.head_groups = (a.batch_heads + 7) / 8;
  a.query_blocks = (int)((S + kQueriesPerBlock - 1) / kQueriesPerBlock);
  a.window = window >= S ? 0 : (int)window;
  if ((int64_t)8 * a.head_groups * a.query_blocks > (int64_t)0x7fffffff)
    return fail(OSLO_E_UNSUPPORTED, "oslo_attention_prefill_fwd: too many blocks for one launch");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == OSLO_F16) return launch_prefill<f16>(a, (int)head_dim, st);
  return launch_prefill<bf16>(a, (int)head_dim, st);
}
} // namespace

extern "C" int oslo_attention_prefill_fwd(void *out, const void *q, const void *k,
                                          const void *v, const float *pad,
                                          float scale, int64_t batch, int64_t heads,
                                          int64_t S, int64_t head_dim,
                                          int64_t window,
                                          const int64_t *strides, int dtype,
                                          oslo_stream_t stream) {
  oslo::DropArgs none{};
  return prefill_entry(out, nullptr, none, q, k, v, pad, scale, batch, heads, S, head_dim,
                       window, strides, dtype, stream);
}

extern "C" int oslo_attention_prefill_fwd_lse(void *out, float *lse, const void *q,
                                              const void *k, const void *v,
                                              const float *pad, float scale, float p,
                                              uint64_t philox_seed,
                                              uint64_t philox_offset, int64_t batch,
                                              int64_t heads, int64_t S,
                                              int64_t head_dim, int64_t window,
                                              const int64_t *strides, int dtype,
                                              oslo_stream_t stream) {
  oslo::DropArgs drop;
  const int s = oslo::make_drop_args("oslo_attention_prefill_fwd_lse", p, philox_seed,
                                     philox_offset, &drop);
  if (s != OSLO_OK) return s;
  if (lse == nullptr && batch > 0 && heads > 0 && S > 0)
    return oslo::fail(OSLO_E_BAD_ARG, "oslo_attention_prefill_fwd_lse: null lse");
  return prefill_entry(out, lse, drop, q, k, v, pad, scale, batch, heads, S, head_dim,
                       window, strides, dtype, stream);
}
