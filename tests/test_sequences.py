"""Sequences of different lengths, the host side: the list of blocks the packed
attention takes its work from, the paged cache's checks, and what the entry
points refuse before they launch anything."""

import ctypes

import numpy as np
import pytest
import torch

from oslo_amd import GPT2Config, GPT2LMHeadModel, GPTNeoConfig, GPTNeoForCausalLM, PackedSequences, PagedKV, PagedState, kernels
from oslo_amd import _lib
from oslo_amd.sequences import packed_labels, sequence_layers


@pytest.mark.parametrize("lengths", [[], [0], [1], [0, 5, 0, 128, 129, 127, 0], [300, 31, 33, 64, 1000]],
                         ids=lambda v: "-".join(map(str, v)) or "none")
def test_blocks_cover_every_token_once(lengths):
    packed = PackedSequences(lengths, "cpu")
    assert packed.total == sum(lengths) and packed.max_length == max(lengths, default=0)
    for which, work in ((0, lambda s, n, b: min(n, 128 * (b + 1))), (1, lambda s, n, b: n - 128 * b)):
        seen = np.zeros(packed.total, dtype=int)
        amounts = []
        for start, n, b, _ in packed.blocks[which].tolist():
            assert 128 * b < n
            seen[start + 128 * b:start + min(n, 128 * (b + 1))] += 1
            amounts.append(work(start, n, b))
        assert (seen == 1).all()
        assert amounts == sorted(amounts, reverse=True)
    assert packed.positions.tolist() == [p for n in lengths for p in range(n)]
    assert packed.sequence.tolist() == [i for i, n in enumerate(lengths) for _ in range(n)]
    assert packed.positions.dtype == torch.int32 and packed.sequence.dtype == torch.int32


def test_shared_blocks_follow_the_work():
    """Blocks are shared where one would outlast the rest of the card, among whole heads of the group."""
    one = PackedSequences([740, 471, 1019, 449, 983, 1387, 4095], "cpu")
    split, parts = one.shared_blocks(32, 8, 128)
    assert parts == 2 and 10 <= split <= 32
    assert one.shared_blocks(32, 32, 128) == (0, 1)                          # no group to share
    assert one.shared_blocks(32, 8, 128, window=64) == (0, 1)                # short walks
    assert PackedSequences([4096] * 16, "cpu").shared_blocks(32, 8, 128) == (0, 1)   # enough blocks of each size
    split, parts = PackedSequences([2000], "cpu").shared_blocks(8, 1, 64)    # 16 blocks on 256 CUs
    assert parts == 8 and split > 8
    assert PackedSequences([], "cpu").shared_blocks(8, 1, 64) == (0, 1)


def test_last_tokens():
    assert PackedSequences([3, 1, 4], "cpu").last_tokens().tolist() == [2, 3, 7]
    with pytest.raises(ValueError):
        PackedSequences([3, 0], "cpu").last_tokens()
    with pytest.raises(ValueError):
        PackedSequences([3, -1], "cpu")
    with pytest.raises(ValueError):
        PackedSequences([2 ** 31], "cpu")


def test_paged_kv_checks_its_tensors():
    pages = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    table = torch.zeros((3, 2), dtype=torch.int32)
    cache = PagedKV(pages, pages.clone(), table)
    assert not cache.quantized and cache.page_size == 16
    with pytest.raises(ValueError):
        PagedKV(pages, pages[:3], table)
    with pytest.raises(ValueError):
        PagedKV(pages, pages.half(), table)
    with pytest.raises(ValueError):
        PagedKV(pages.float(), pages.float(), table)
    with pytest.raises(ValueError):
        PagedKV(pages.transpose(1, 2), pages.transpose(1, 2), table)
    with pytest.raises(ValueError):
        PagedKV(pages, pages.clone(), table.long())
    with pytest.raises(ValueError):
        PagedKV(pages, pages.clone(), table, torch.zeros((4, 2, 16), dtype=torch.uint8),
                torch.zeros((4, 2, 16), dtype=torch.uint8))
    eight = pages.to(torch.float8_e4m3fn)
    scales = torch.full((4, 2, 16), 127, dtype=torch.uint8)
    assert PagedKV(eight, eight.clone(), table, scales, scales.clone()).quantized
    with pytest.raises(ValueError):
        PagedKV(eight, eight.clone(), table)
    with pytest.raises(ValueError):
        PagedKV(eight, eight.clone(), table, scales, scales[:, :1])


def test_operators_reject_host_tensors():
    q = torch.zeros((4, 2, 64), dtype=torch.bfloat16)
    packed = PackedSequences([4], "cpu")
    table = torch.zeros((4, 1), dtype=torch.int32)
    pages = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    cache = PagedKV(pages, pages.clone(), table)
    index = torch.zeros(4, dtype=torch.int32)
    for call in (lambda: kernels.attention_packed_forward(q, q, q, packed, 1.0),
                 lambda: kernels.paged_kv_write(cache, q, q, index, index),
                 lambda: kernels.paged_kv_read(cache, index, index, torch.bfloat16),
                 lambda: kernels.attention_paged_decode_forward(q, cache, index, 1.0),
                 lambda: kernels.sample_forward(torch.zeros((2, 8)), torch.zeros(2))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_entry_points_screen_their_arguments():
    """Every call here fails, or has nothing to do, before any pointer is followed."""
    lib = _lib.load()
    null, one, odd = ctypes.c_void_p(0), ctypes.c_void_p(16), ctypes.c_void_p(24)

    def strides(*pairs):
        return (ctypes.c_int64 * len(pairs))(*pairs)

    # packed attention: 40 tokens, 4 heads on 2, 64 features
    good = strides(64, 256, 64, 128, 64, 128, 64, 256)

    def packed(blocks=one, n=1, scale=0.125, tokens=40, longest=40, heads=4, kv=2, d=64, window=0, st=good, dtype=2,
               out=one, q=one):
        return lib.oslo_attention_packed_fwd(out, null, null, q, one, one, blocks, n, scale, tokens, longest, heads, kv, d,
                                             window, st, dtype, null)
    assert packed(n=-1) == -1 and packed(tokens=-1) == -1 and packed(window=-1) == -1
    assert packed(dtype=0) == -2 and packed(dtype=7) == -1
    assert packed(d=48) == -2
    assert packed(scale=0.0) == -1 and packed(scale=float("nan")) == -1
    assert packed(heads=5) == -1 and packed(kv=0) == -1
    assert b"share" in lib.oslo_last_error()
    assert packed(longest=41) == -1 and packed(longest=0) == -1
    assert packed(blocks=null) == -1 and packed(q=null) == -1 and packed(out=odd) == -2
    assert packed(st=strides(64, 256, 64, 128, 64, 128, 64, 32)) == -2      # token stride below head_dim
    assert packed(st=strides(64, 260, 64, 128, 64, 128, 64, 256)) == -2     # not a multiple of 8
    assert packed(st=strides(64, 2 ** 30, 64, 128, 64, 128, 64, 256)) == -2  # a sequence of a head over 2 GiB
    assert packed(tokens=2 ** 31, longest=40) == -2
    assert packed(heads=2 ** 17, kv=1, st=good) == -2
    assert packed(n=0) == 0 and packed(tokens=0) == 0 and packed(heads=0, kv=0) == 0
    assert lib.oslo_attention_packed_bwd_workspace_bytes(40, 4, 2, 64, 0, 1) == 640
    assert lib.oslo_attention_packed_bwd_workspace_bytes(0, 4, 2, 64, 0, 1) == 0
    assert lib.oslo_attention_packed_bwd_workspace_bytes(41, 3, 1, 64, 2, 3) == (124 + 2 * 3 * 2 * 128 * 64) * 4
    good16 = strides(*(list(good[:8]) + [64, 256, 64, 256, 64, 128, 64, 128]))

    def packed_bwd(ws=one, keys=one, lse=one, dq=one, split=0, parts=1):
        return lib.oslo_attention_packed_bwd(dq, one, one, one, one, one, one, one, null, lse, ws, one, keys, 1, split, parts, 0.125, 40, 40,
                                             4, 2, 64, 0, good16, 2, null)
    assert packed_bwd(ws=null) == -1 and packed_bwd(keys=null) == -1 and packed_bwd(lse=null) == -1
    assert packed_bwd(ws=odd) == -2 and packed_bwd(dq=odd) == -2
    assert packed_bwd(split=2) == -1 and packed_bwd(split=1, parts=3) == -1 and packed_bwd(parts=0) == -1

    # paged cache: 3 sequences of 5 pages, a pool of 20, 2 heads, pages of 16, 64 features
    st4 = strides(64, 128, 64, 128)

    def write(kp=one, vp=one, ks=null, vs=null, k=one, seq=one, table=one, tokens=7, page=16, d=64, dtype=2, st=st4,
              max_pages=5):
        return lib.oslo_paged_kv_write(kp, vp, ks, vs, k, one, seq, one, table, tokens, 3, max_pages, 20, 2, page, d,
                                       st, dtype, null)
    assert write(tokens=-1) == -1 and write(page=24) == -2 and write(page=8) == -2 and write(page=8192) == -2
    assert write(d=80) == -2 and write(dtype=0) == -2 and write(dtype=9) == -1
    assert write(ks=one) == -1 and b"together" in lib.oslo_last_error()
    assert write(kp=null) == -1 and write(table=null) == -1 and write(k=null) == -1 and write(seq=null) == -1
    assert write(kp=odd) == -2 and write(k=odd) == -2 and write(ks=odd, vs=one) == -2
    assert write(st=strides(60, 128, 64, 128)) == -2 and write(st=None) == -1
    assert write(max_pages=2 ** 26) == -2
    assert write(tokens=0) == 0
    assert lib.oslo_paged_kv_read(null, one, one, one, null, null, one, one, one, 7, 3, 5, 20, 2, 16, 64, 2, null) == -1
    assert lib.oslo_paged_kv_read(one, one, one, one, null, null, one, one, one, 0, 3, 5, 20, 2, 16, 64, 2, null) == 0

    def decode(out=one, q=one, lengths=one, ws=one, scale=0.125, seqs=3, heads=4, kv=2, window=0, dtype=2, d=64,
               max_pages=5, num_pages=20, st=strides(64, 256)):
        return lib.oslo_attention_paged_decode_fwd(out, q, one, one, null, null, one, lengths, ws, scale, seqs,
                                                   max_pages, num_pages, heads, kv, 16, d, window, st, dtype, null)
    assert decode(heads=-1) == -1 and decode(window=-1) == -1 and decode(scale=-1.0) == -1
    assert decode(heads=5) == -1 and decode(dtype=0) == -2 and decode(d=32) == -2
    assert decode(lengths=null) == -1 and decode(out=odd) == -2 and decode(st=strides(4, 256)) == -2
    assert decode(max_pages=0) == -1 and decode(num_pages=0) == -1
    assert decode(max_pages=4096, ws=null) == -1 and b"workspace" in lib.oslo_last_error()
    assert decode(seqs=0) == 0 and decode(heads=0) == 0
    assert lib.oslo_attention_paged_decode_workspace_bytes(3, 5, 2, 64, 4096, 0) == 0

    # sampling
    def sample(tokens=one, logits=one, t=1.0, k=0, p=1.0, m=0.0, rows=2, vocab=50, dtype=0):
        return lib.oslo_sample(tokens, null, logits, one, null, t, null, k, null, p, null, m, rows, vocab, vocab, dtype,
                               null)
    assert sample(t=-0.5) == -1 and sample(t=float("nan")) == -1 and sample(k=-1) == -1
    assert sample(p=-0.1) == -1 and sample(m=1.5) == -1 and sample(m=-0.1) == -1
    assert sample(vocab=0) == -1 and sample(vocab=2 ** 24 + 1) == -2 and sample(rows=-1) == -1
    assert sample(dtype=5) == -1 and sample(tokens=null) == -1 and sample(logits=null) == -1
    assert sample(rows=0) == 0


def test_labels_of_a_packed_row_stay_inside_their_sequences():
    """Next tokens; none at a sequence's end, behind the last sequence, or where the caller has none."""
    packed = PackedSequences([3, 0, 1, 4], "cpu")
    labels = torch.tensor([[10, 11, 12, 20, 30, 31, -100, 33, 98, 99]])
    assert packed_labels(labels, packed).tolist() == [[11, 12, -100, -100, 31, -100, 33, -100, -100, -100]]
    assert packed_labels(labels[:, :1], PackedSequences([1], "cpu")).tolist() == [[-100]]
    assert packed_labels(labels[:, :0], PackedSequences([], "cpu")).tolist() == [[]]


def test_positions_of_a_row_with_tokens_behind_the_last_sequence():
    layer = sequence_layers(PackedSequences([2, 3], "cpu"), 1)[0]
    assert layer.row_positions(5).tolist() == [0, 1, 0, 1, 2]
    assert layer.row_positions(7).tolist() == [0, 1, 0, 1, 2, 0, 0]
    with pytest.raises(ValueError, match="5 tokens of sequences in a row of 4"):
        layer.row_positions(4)


def test_paged_state_gives_every_sequence_its_own_pages_and_stops_at_the_last_position():
    state = PagedState([3, 130, 0], 131, 2, 2, 64, torch.float16, "cpu")
    assert state.table.shape == (3, 3) and sorted(state.table.flatten().tolist()) == list(range(9))
    assert len(state.caches) == 2 and all(c.key_pages.shape == (9, 2, 64, 64) for c in state.caches)
    layers = state.begin_step()
    assert state.visible.tolist() == [4, 131, 1] and layers[1].positions is state.lengths
    state.end_step()
    assert state.lengths.tolist() == [4, 130, 1]
    for bad in (dict(lengths=[5], capacity=4), dict(lengths=[-1], capacity=4), dict(lengths=[0], capacity=0)):
        with pytest.raises(ValueError, match="PagedState"):
            PagedState(**bad, layers=1, kv_heads=1, head_dim=64, dtype=torch.float16, device="cpu")


def test_a_sequence_that_is_full_from_the_start_stays_at_its_last_position():
    """Prompts of as many tokens as there are positions: the fed token's position, and what it sees, stay inside."""
    from oslo_amd.modeling_gptj import rotary_for_step
    state = PagedState([4, 2, 4], 4, 1, 1, 64, torch.float16, "cpu", page_size=16)
    for _ in range(2):
        layer = state.begin_step()[0]
        assert layer.positions.tolist()[::2] == [3, 3] and int(state.visible.max()) <= state.capacity
        sin, cos, offset = rotary_for_step(layer, 64, 3, torch.device("cpu"))
        assert sin.shape == cos.shape == (3, 32) and offset == 0
        state.end_step()
    assert state.lengths.tolist() == [3, 3, 3]


def test_rotary_tables_live_as_long_as_what_reads_them():
    """A captured step goes on reading its tables, whatever other lengths are asked for in between."""
    import weakref

    from oslo_amd import DecodeState, StaticKV
    from oslo_amd import modeling_gptj as gptj
    state = PagedState([4, 2], 37, 1, 1, 64, torch.float16, "cpu", page_size=16)
    packed = PackedSequences([29, 3], "cpu")
    static = DecodeState(41, "cpu", torch.float16)
    layers = [(state.begin_step()[0], 2), (sequence_layers(packed, 1)[0], 32),
              (StaticKV(static, *(torch.zeros((1, 1, 41, 64)) for _ in range(2))), 1)]
    device = torch.device("cpu")
    tables = []
    for (layer, n), positions in zip(layers, (37, 29, 41)):
        gptj.rotary_for_step(layer, 32, n, device)
        tables.append([weakref.ref(t) for t in gptj.rotary_tables(32, positions, device)])
    del layer, layers
    for n in range(50, 70):
        gptj.rotary_tables(32, n, device)
    for holder, refs in zip((state, packed, static), tables):
        assert all(r() is not None for r in refs)
    del state, packed, static, holder
    import gc
    gc.collect()
    assert all(r() is None for refs in tables for r in refs)


def test_tangents_of_forward_mode_are_not_dropped():
    """A dual tensor needs no ``requires_grad``, and ``no_grad`` does not turn it off: torch carries the tangent on
    through both, so an operator without one has to say so."""
    from torch.autograd import forward_ad

    from oslo_amd import FusedPagedDecodeAttention, FusedPagedKV
    from oslo_amd.fused_kernels_utils import _needs_grad
    x = torch.zeros((4, 2, 64), dtype=torch.bfloat16)
    pages = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    cache = PagedKV(pages, pages.clone(), torch.zeros((4, 1), dtype=torch.int32))
    index = torch.zeros(4, dtype=torch.int32)
    assert not _needs_grad(x, None)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        assert not _needs_grad(x, None)
        for mode in (torch.enable_grad, torch.no_grad):
            with mode():
                assert _needs_grad(x, None, dual) and forward_ad.unpack_dual(dual * 2).tangent is not None
                for call in (lambda: FusedPagedKV.write(cache, x, dual, index, index),
                             lambda: FusedPagedDecodeAttention.apply(dual, cache, index)):
                    with pytest.raises(RuntimeError, match="tangent"):
                        call()
    assert not _needs_grad(x)


def test_packed_sequences_are_whole_once_they_are_made(monkeypatch):
    """Nothing is copied from the host later (a capture allows no such copy): positions, owners and last tokens too."""
    packed = PackedSequences([3, 1, 4], "cpu")

    def refuse(*args, **kwargs):
        raise AssertionError("made from host data")
    monkeypatch.setattr(torch, "from_numpy", refuse)
    monkeypatch.setattr(torch, "tensor", refuse)
    assert packed.positions.tolist() == [0, 1, 2, 0, 0, 1, 2, 3] and packed.sequence.tolist() == [0, 0, 0, 1, 2, 2, 2, 2]
    last = packed.last_tokens()
    assert last.tolist() == [2, 3, 7] and last.dtype == torch.int64
    assert packed.blocks.is_contiguous() and packed.blocks.tolist()[0] == [[4, 4, 0, 0], [0, 3, 0, 0], [3, 1, 0, 0]]
    assert sequence_layers(packed, 1)[0].row_positions(9).tolist() == [0, 1, 2, 0, 0, 1, 2, 3, 0]


def test_prompts_that_a_state_has_no_place_for_are_refused():
    """The cache passes over tokens that name no place of it: prompts would be cut without a word."""
    state = PagedState([4, 2], 8, 3, 1, 64, torch.float16, "cpu", page_size=16)
    for bad in ([4, 2, 1], [9, 2], [16, 1]):
        with pytest.raises(ValueError, match="places for 2 of up to 8"):
            state.prompt_layers(PackedSequences(bad, "cpu"))
    for good in ([4, 2], [8, 8], [3], []):
        assert len(state.prompt_layers(PackedSequences(good, "cpu"))) == 3


def test_leaves_behind_views_are_looked_at(monkeypatch):
    """The slices of one leaf, as an attention's query, key and value are."""
    from oslo_amd.fused_kernels_utils import _check_captured_leaves
    capturing = [False]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    leaf, other = (torch.ones((6, 12), requires_grad=True) for _ in range(2))

    def result(x):
        q, k, v = x.view(6, 3, 4).unbind(1)
        return torch.stack([q, k.contiguous(), v.t().t()])
    living = result(leaf)
    _check_captured_leaves(living)
    capturing[0] = True
    with pytest.raises(RuntimeError, match="eager graph of the same leaf"):
        _check_captured_leaves(result(leaf))
    _check_captured_leaves(result(other))
    _check_captured_leaves(result(leaf + other))  # (of two inputs: not followed)
    del living
    _check_captured_leaves(result(leaf))


def test_models_refuse_what_sequences_do_not_take():
    model = GPT2LMHeadModel(GPT2Config(vocab_size=11, n_positions=8, n_embd=64, n_layer=1, n_head=1)).eval()
    row, packed = torch.zeros((1, 6), dtype=torch.long), PackedSequences([2, 4], "cpu")
    with pytest.raises(RuntimeError, match="fuse"):
        model(row, packed=packed)
    with pytest.raises(ValueError, match="without past_key_values"):
        model(row, packed=packed, use_cache=True)
    with pytest.raises(ValueError, match="without past_key_values"):
        model(row, packed=packed, attention_mask=torch.ones_like(row))
    model.fuse()
    with pytest.raises(ValueError, match="one row"):
        model(row.view(2, 3), packed=packed)
    with pytest.raises(ValueError, match="the model has 8"):
        model(torch.zeros((1, 9), dtype=torch.long), packed=PackedSequences([9], "cpu"))
    with pytest.raises(ValueError, match="6 tokens of sequences in a row of 5"):
        model(row[:, :5], packed=packed)
    with pytest.raises(RuntimeError, match="drop"):
        model.train()(row, packed=packed)
    from oslo_amd.modeling_gpt_neo import GPTNeoSelfAttention
    half = GPTNeoForCausalLM(GPTNeoConfig(vocab_size=11, max_position_embeddings=8, hidden_size=64, num_layers=2, num_heads=1))
    half.fuse(modules=[GPTNeoSelfAttention])  # (its local layers are not)
    with pytest.raises(RuntimeError, match="fuse"):
        half.eval()(row, packed=packed)


def test_generate_refuses_what_sampling_and_lists_do_not_take():
    model = GPT2LMHeadModel(GPT2Config(vocab_size=11, n_positions=8, n_embd=64, n_layer=1, n_head=1)).eval()
    ids = torch.zeros((1, 3), dtype=torch.long)
    with pytest.raises(ValueError, match="num_beams=1"):
        model.generate(ids, max_length=5, do_sample=True, num_beams=2)
    with pytest.raises(ValueError, match="list of prompts"):
        model.generate(ids, max_length=5, quantized_cache=True)
    for kw in (dict(num_beams=2), dict(no_repeat_ngram_size=2), dict(static_cache=True), dict(use_cache=False)):
        with pytest.raises(ValueError, match="its own paged cache"):
            model.generate([ids[0]], max_length=5, **kw)
    for bad in ([ids], [ids[0, :0]], [ids[0].repeat(2)]):
        with pytest.raises(ValueError, match="1-D tensors of 1 to max_length - 1 = 4"):
            model.generate(bad, max_length=5)
    with pytest.raises(RuntimeError, match="ROCm device"):
        model.generate([ids[0]], max_length=5)
    assert model.generate([], max_length=5) == []


def test_decode_workspace_fits_every_launch_of_a_call():
    """A call of more sequences than one launch takes (4096) ends with a smaller launch, which must not want more
    than the call's workspace; what kind of launch it is goes by the whole call."""
    need = _lib.load().oslo_attention_paged_decode_workspace_bytes
    for heads, kv_heads, d in ((1, 1, 64), (2, 1, 128), (8, 8, 256), (34, 2, 64)):
        for length in (32, 64, 256, 512, 528, 1024, 1040, 4096, 131072):
            for window in (0, 40, 700):
                whole = need(4097, heads, kv_heads, d, length, window)
                assert whole == need(4096, heads, kv_heads, d, length, window)
                if whole:
                    assert max(need(n, heads, kv_heads, d, length, window) for n in range(1, 4096, 7)) <= whole
