// Backward of the attention over packed sequences (attention_packed.hip): the
// passes of the prompt attention's backward (attention_prefill_bwd.hpp) on the
// list of blocks. The pass for dQ takes 128 queries of one query head; the
// passes for dK and dV take 128 keys of one key/value head and walk the queries
// of every head of its group, so the sum over the group is formed in the fp32
// accumulators, in a fixed order, and rounded once. No [S, S] tile is kept in
// memory at any head size. Two lists of the same entries: the dQ pass wants the
// blocks with the most keys first, the others those with the most queries left.

#include "attention_packed.hpp"
#include "attention_prefill_bwd.hpp"

namespace oslo {
namespace {

static_assert(kOwnPerBlock == kPackedPositions, "an entry of the list is a block of the kernel");

template <typename T, int D, int ROLE>
int launch_packed_role(const BwdArgs &a, int64_t num_blocks, hipStream_t stream) {
  constexpr unsigned kLds = sched_lds_bytes<T, D, ROLE>();
  auto *kernel = a.window > 0 ? attention_bwd_kernel<T, D, ROLE, false, true, false, false, true>
                              : attention_bwd_kernel<T, D, ROLE, false, false, false, false, true>;
  if (kLds > 64u * 1024u) {
    const int s = raise_lds_limit(reinterpret_cast<const void *>(kernel), kLds, "oslo_attention_packed_bwd");
    if (s != OSLO_OK) return s;
  }
  const int64_t heads = ROLE == kRoleDQ ? a.heads : a.packed.kv_heads;
  kernel<<<dim3((unsigned)(num_blocks * heads)), dim3(kBlockThreads), kLds, stream>>>(a);
  return check_launch("attention_packed_bwd");
}

template <typename T, int D>
int launch_packed_bwd(BwdArgs a, const int32_t *query_blocks, const int32_t *key_blocks, int64_t num_blocks,
                      float *delta, const void *out, const Strides3 &so, hipStream_t stream) {
  const int64_t rows = (int64_t)a.heads * a.packed.tokens;
  constexpr int kRows = kBlockThreads / (D / 8);
  attention_delta_kernel<T, D><<<dim3((unsigned)((rows + kRows - 1) / kRows)), dim3(kBlockThreads), 0, stream>>>(
      delta, static_cast<const T *>(out), static_cast<const T *>(a.dout), so, a.sdo, (int)a.packed.tokens, a.heads,
      rows);
  int s = check_launch("attention_packed_bwd(delta)");
  if (s != OSLO_OK) return s;
  a.packed.blocks = query_blocks;
  s = launch_packed_role<T, D, kRoleDQ>(a, num_blocks, stream);
  if (s != OSLO_OK) return s;
  a.packed.blocks = key_blocks;
  // (one pass for both where the accumulators fit a lane's registers, as in the dense backward)
  if constexpr (D <= 128) {
    return launch_packed_role<T, D, kRoleDKV>(a, num_blocks, stream);
  } else {
    s = launch_packed_role<T, D, kRoleDK>(a, num_blocks, stream);
    if (s != OSLO_OK) return s;
    return launch_packed_role<T, D, kRoleDV>(a, num_blocks, stream);
  }
}

template <typename T>
int launch_packed_bwd_dim(const BwdArgs &a, const int32_t *query_blocks, const int32_t *key_blocks, int64_t num_blocks,
                          float *delta, const void *out, const Strides3 &so, int64_t head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 64: return launch_packed_bwd<T, 64>(a, query_blocks, key_blocks, num_blocks, delta, out, so, stream);
    case 128: return launch_packed_bwd<T, 128>(a, query_blocks, key_blocks, num_blocks, delta, out, so, stream);
    default: return launch_packed_bwd<T, 256>(a, query_blocks, key_blocks, num_blocks, delta, out, so, stream);
  }
}

} // namespace
} // namespace oslo

extern "C" size_t oslo_attention_packed_bwd_workspace_bytes(int64_t tokens, int64_t heads) {
  if (tokens <= 0 || heads <= 0) return 0;
  return (size_t)tokens * (size_t)heads * sizeof(float);
}

extern "C" int oslo_attention_packed_bwd(void *dq, void *dk, void *dv, const void *dout, const void *q,
                                         const void *k, const void *v, const void *out,
                                         const float *lse, float *workspace,
                                         const int32_t *query_blocks,
                                         const int32_t *key_blocks, int64_t num_blocks,
                                         float scale, int64_t tokens, int64_t max_length,
                                         int64_t heads, int64_t kv_heads, int64_t head_dim,
                                         int64_t window, const int64_t *strides, int dtype,
                                         oslo_stream_t stream) {
  using namespace oslo;
  const char *const name = "oslo_attention_packed_bwd";
  const void *tensors[8] = {q, k, v, out, dout, dq, dk, dv};
  const int s = check_packed(name, tensors, strides, 8, scale, query_blocks, num_blocks, tokens, max_length, heads,
                             kv_heads, head_dim, window, dtype);
  if (s != OSLO_OK) return s;
  if (num_blocks == 0 || heads == 0 || tokens == 0) return OSLO_OK;
  if (!key_blocks || !lse || !workspace) return fail(OSLO_E_BAD_ARG, "%s: null pointer", name);
  if (!aligned16(lse) || !aligned16(workspace))
    return fail(OSLO_E_UNSUPPORTED, "%s: lse and the workspace must be 16-byte aligned", name);
  if (heads * tokens > (int64_t)0x7fffffff)
    return fail(OSLO_E_UNSUPPORTED, "%s: too many rows for one launch", name);
  auto st = [&](int i) { return Strides3{0, strides[2 * i], strides[2 * i + 1]}; };
  BwdArgs a{};
  a.q = q, a.k = k, a.v = v, a.dout = dout, a.dq = dq, a.dk = dk, a.dv = dv;
  a.lse = lse, a.delta = workspace;
  a.sq = st(0), a.sk = st(1), a.sv = st(2), a.sdo = st(4), a.sdq = st(5), a.sdk = st(6), a.sdv = st(7);
  a.scale = scale;
  a.scale_log2e = scale * kLog2eB;
  a.heads = (int)heads;
  a.window = window >= max_length ? 0 : (int)window;
  a.packed = packed_args(query_blocks, tokens, max_length, heads, kv_heads);
  hipStream_t stm = static_cast<hipStream_t>(stream);
  if (dtype == OSLO_F16)
    return launch_packed_bwd_dim<f16>(a, query_blocks, key_blocks, num_blocks, workspace, out, st(3), head_dim, stm);
  return launch_packed_bwd_dim<bf16>(a, query_blocks, key_blocks, num_blocks, workspace, out, st(3), head_dim, stm);
}
