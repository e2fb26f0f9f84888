// Backward of the attention over packed sequences (attention_packed.hip): the
// passes of the prompt attention's backward (attention_prefill_bwd.hpp) on the
// list of blocks. The pass for dQ takes 128 queries of one query head; the
// passes for dK and dV take 128 keys of one key/value head and walk the queries
// of every head of its group, so the sum over the group is formed in the fp32
// accumulators, in a fixed order, and rounded once. No [S, S] tile is kept in
// memory at any head size.
//
// A block's walk grows with the group: at 4 query heads per key/value head and one
// sequence of 4095 tokens among 9144, its first keys meet 4 x 4095 queries, 1.4 times
// what a CU does on average, and the rest of the card waits for that block. So the
// caller may have the first entries of the list (those with most queries) shared by
// several blocks, each with some heads of the group, whose fp32 sums a last kernel
// adds in order: 575 us become 460 to 500 for the dK/dV pass there (355 Gflop, 0.74
// Pflop/s), and 9 us go into the last kernel; the dQ pass takes 295 (267 Gflop, 0.9).
// With a window of 256 (8794 tokens, 20 heads) the passes take 84 and 137 us, half of it
// for what a block reads and writes before and after its 12 tiles: 7.9 us a tile over
// both passes, 112 us for the rest, which at one block per CU of the pass for dK and dV nothing hides.
// At 256 features every pass computes the scores anew, 8 products a tile where the dense backward's tile
// store makes it 5: 16 heads, 8 sequences of 2048 tokens 1328 us (dense 1064), 8 of 1024 423 (327), the 9
// prompts of 8299 tokens 493.
//
// Two lists of the same entries: the dQ pass wants the blocks with the most keys first,
// the others those with the most queries left.

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
  const int64_t entries = ROLE == kRoleDQ ? num_blocks : num_blocks + (int64_t)a.split * (a.parts - 1);
  kernel<<<dim3((unsigned)(entries * heads)), dim3(kBlockThreads), kLds, stream>>>(a);
  return check_launch("attention_packed_bwd");
}

// dK and dV of the entries whose group was shared: the sum over the parts, in order.
// A thread per four features.
template <typename T, int D>
__global__ __launch_bounds__(kBlockThreads) void attention_packed_join_kernel(const BwdArgs a) {
  constexpr int kRowThreads = D / 4, kRows = kBlockThreads / kRowThreads;
  const int share = threadIdx.x % kRowThreads;
  unsigned index = blockIdx.x;
  const int row = (int)(index % (kOwnPerBlock / kRows)) * kRows + threadIdx.x / kRowThreads;
  index /= kOwnPerBlock / kRows;
  const int which = (int)(index & 1u);
  index >>= 1;
  const int kv_head = (int)(index % (unsigned)a.packed.kv_heads);
  const unsigned entry = index / (unsigned)a.packed.kv_heads;
  const PackedBlock e = packed_block(a.packed, entry);
  if (!packed_block_in_range(a.packed, e, kOwnPerBlock)) return;
  const int position = e.block * kOwnPerBlock + row;
  if (position >= e.length) return;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p = 0; p < a.parts; ++p) {
    const int64_t slot = ((int64_t)entry * a.parts + p) * a.packed.kv_heads + kv_head;
    const float4 v = *reinterpret_cast<const float4 *>(a.partial + ((slot * 2 + which) * kOwnPerBlock + row) * D + 4 * share);
    sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
  }
  const Strides3 &st = which ? a.sdv : a.sdk;
  typedef T Out4 __attribute__((ext_vector_type(4)));
  Out4 w;
  w[0] = static_cast<T>(sum.x), w[1] = static_cast<T>(sum.y), w[2] = static_cast<T>(sum.z), w[3] = static_cast<T>(sum.w);
  *reinterpret_cast<Out4 *>(static_cast<T *>(which ? a.dv : a.dk) + kv_head * st.h + (e.start + position) * st.s + 4 * share) = w;
}

template <typename T, int D>
int launch_packed_bwd(BwdArgs a, const int32_t *query_blocks, const int32_t *key_blocks, int64_t num_blocks,
                      hipStream_t stream) {
  a.packed.blocks = query_blocks;
  int s = launch_packed_role<T, D, kRoleDQ>(a, num_blocks, stream);
  if (s != OSLO_OK) return s;
  a.packed.blocks = key_blocks;
  // (one pass for both where the accumulators fit a lane's registers, as in the dense backward)
  if constexpr (D <= 128) {
    s = launch_packed_role<T, D, kRoleDKV>(a, num_blocks, stream);
  } else {
    s = launch_packed_role<T, D, kRoleDK>(a, num_blocks, stream);
    if (s != OSLO_OK) return s;
    s = launch_packed_role<T, D, kRoleDV>(a, num_blocks, stream);
  }
  if (s != OSLO_OK || a.split == 0) return s;
  constexpr int kRows = kBlockThreads / (D / 4);
  attention_packed_join_kernel<T, D><<<dim3((unsigned)((int64_t)a.split * a.packed.kv_heads * 2 * (kOwnPerBlock / kRows))),
                                       dim3(kBlockThreads), 0, stream>>>(a);
  return check_launch("attention_packed_bwd(join)");
}

template <typename T>
int launch_packed_bwd_dim(const BwdArgs &a, const int32_t *query_blocks, const int32_t *key_blocks, int64_t num_blocks,
                          int64_t head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 64: return launch_packed_bwd<T, 64>(a, query_blocks, key_blocks, num_blocks, stream);
    case 128: return launch_packed_bwd<T, 128>(a, query_blocks, key_blocks, num_blocks, stream);
    default: return launch_packed_bwd<T, 256>(a, query_blocks, key_blocks, num_blocks, stream);
  }
}

} // namespace
} // namespace oslo

extern "C" size_t oslo_attention_packed_bwd_workspace_bytes(int64_t tokens, int64_t heads, int64_t kv_heads,
                                                            int64_t head_dim, int64_t split, int64_t parts) {
  if (tokens <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || split < 0 || parts < 1) return 0;
  const size_t rows = ((size_t)tokens * (size_t)heads + 3) / 4 * 4;
  return (rows + (size_t)split * (size_t)(split ? parts : 0) * (size_t)kv_heads * 2 * oslo::kOwnPerBlock *
                     (size_t)head_dim) * sizeof(float);
}

extern "C" int oslo_attention_packed_bwd(void *dq, void *dk, void *dv, const void *dout, const void *q,
                                         const void *k, const void *v, const void *out,
                                         const void *out_low,
                                         const float *lse, float *workspace,
                                         const int32_t *query_blocks,
                                         const int32_t *key_blocks, int64_t num_blocks,
                                         int64_t split, int64_t parts,
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
  if (split < 0 || split > num_blocks || parts < 1 || (split > 0 && kv_heads > 0 && parts > heads / kv_heads))
    return fail(OSLO_E_BAD_ARG, "%s: %lld entries shared by %lld blocks each", name, (long long)split, (long long)parts);
  if (num_blocks == 0 || heads == 0 || tokens == 0) return OSLO_OK;
  if (!key_blocks || !lse || !workspace) return fail(OSLO_E_BAD_ARG, "%s: null pointer", name);
  if (!aligned16(lse) || !aligned16(workspace) || !aligned16(out_low))
    return fail(OSLO_E_UNSUPPORTED, "%s: out_low, lse and the workspace must be 16-byte aligned", name);
  if (heads * tokens > (int64_t)0x7fffffff || (num_blocks + split * parts) > (int64_t)0x7fffffff / (heads * 64))
    return fail(OSLO_E_UNSUPPORTED, "%s: too many rows for one launch", name);
  auto st = [&](int i) { return Strides3{0, strides[2 * i], strides[2 * i + 1]}; };
  BwdArgs a{};
  a.q = q, a.k = k, a.v = v, a.dout = dout, a.dq = dq, a.dk = dk, a.dv = dv, a.out = out, a.out_low = out_low;
  a.lse = lse, a.delta = a.delta_out = workspace;
  a.partial = workspace + (heads * tokens + 3) / 4 * 4;
  a.split = (int)split, a.parts = (int)parts;
  a.sq = st(0), a.sk = st(1), a.sv = st(2), a.sout = st(3), a.sdo = st(4), a.sdq = st(5), a.sdk = st(6), a.sdv = st(7);
  a.scale = scale;
  a.scale_log2e = scale * kLog2eB;
  a.heads = (int)heads;
  a.window = window >= max_length ? 0 : (int)window;
  a.packed = packed_args(query_blocks, tokens, max_length, heads, kv_heads);
  hipStream_t stm = static_cast<hipStream_t>(stream);
  if (dtype == OSLO_F16) return launch_packed_bwd_dim<f16>(a, query_blocks, key_blocks, num_blocks, head_dim, stm);
  return launch_packed_bwd_dim<bf16>(a, query_blocks, key_blocks, num_blocks, head_dim, stm);
}
