"""The paged key/value cache (written in 16 or 8 bits, read back) and the
attention of one new token per sequence over it, against plain code in float64.

Tolerances. 16-bit copies and the 8-bit storage are exact (the storage is
compared with a scale and a rounding worked out here). The attention reads exact
values, rounds each probability to 16 bits before it multiplies v and the result
once: with REL half a step of the type, REL * (P |v|) + REL * |out|, taken 1.05
times, plus 2^-15 of P |v| for the fp32 scores, exponentials and sums. The
chunks' join adds fp32 products, within the same 2^-15."""

import math

import pytest
import torch

from oslo_amd import FusedPagedDecodeAttention, FusedPagedKV, PagedKV
from tests.util import IDS, randn

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
REL = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
HALVES = [torch.float16, torch.bfloat16]


def make_table(pages_of, order_seed=0):
    """Pages handed out in shuffled order, three of the pool left unused."""
    total = sum(pages_of) + 3
    order = torch.randperm(total, generator=torch.Generator().manual_seed(order_seed)).tolist()
    table = torch.zeros((len(pages_of), max(max(pages_of), 1)), dtype=torch.int32)
    at = 0
    for i, n in enumerate(pages_of):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return table, total


def poisoned(lengths, kv_heads, d, page, dtype, eight, seed=0):
    """A cache in which every place holds NaN (and, in 8 bits, the largest scale byte)."""
    table, total = make_table([-(-n // page) for n in lengths], seed)
    shape = (total, kv_heads, page, d)
    if eight:
        pages = [torch.full(shape, 0x7f, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2)]
        return PagedKV(*pages, table.to(DEV), *(torch.full(shape[:3], 255, dtype=torch.uint8, device=DEV) for _ in range(2)))
    pages = [torch.full(shape, float("nan"), dtype=dtype, device=DEV) for _ in range(2)]
    return PagedKV(*pages, table.to(DEV))


def tokens_of(lengths):
    seq = [i for i, n in enumerate(lengths) for _ in range(n)]
    pos = [p for n in lengths for p in range(n)]
    return (torch.tensor(seq, dtype=torch.int32, device=DEV), torch.tensor(pos, dtype=torch.int32, device=DEV))


def stored(x):
    """What 8-bit storage keeps of x [.., D], in float64 on the CPU: the least power of
    two that brings the largest finite magnitude to 448 or below, and the nearest
    multiple of each value's step (ties to even)."""
    x = x.double().cpu()
    finite = torch.isfinite(x)
    amax = torch.where(finite, x.abs(), torch.zeros_like(x)).amax(-1, keepdim=True)
    e = torch.zeros_like(amax)
    some = amax > 0
    e[some] = torch.ceil(torch.log2(amax[some] / 448.0))
    e = torch.where(some & (amax > 448.0 * 2.0 ** e), e + 1, e)
    e = torch.where(some & (amax <= 448.0 * 2.0 ** (e - 1)), e - 1, e)
    e = e.clamp(min=-126.0)
    y = x / 2.0 ** e
    size = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -20))).clamp(-6.0, 8.0)
    step = 2.0 ** (size - 3)
    return torch.where(finite, torch.round(y / step) * step * 2.0 ** e, torch.full_like(x, math.nan))


@pytest.mark.parametrize("dtype", HALVES, ids=IDS.get)
@pytest.mark.parametrize("eight", [False, True], ids=["16bit", "8bit"])
@pytest.mark.parametrize("lengths,kv_heads,d,page", [([1], 1, 64, 16), ([33, 0, 5, 129], 3, 128, 16),
                                                     ([70, 64, 1], 12, 64, 32), ([300, 17], 2, 256, 128)],
                         ids=lambda v: str(v).replace(" ", ""))
def test_write_then_read(lengths, kv_heads, d, page, eight, dtype):
    cache = poisoned(lengths, kv_heads, d, page, dtype, eight)
    seq, pos = tokens_of(lengths)
    t = len(seq)
    k, v = (randn((t, kv_heads, d), dtype, seed=s, std=3.0).to(DEV) for s in (1, 2))
    shuffle = torch.randperm(t, generator=torch.Generator().manual_seed(4)).to(DEV)
    FusedPagedKV.write(cache, k[shuffle], v[shuffle], seq[shuffle], pos[shuffle])
    back = FusedPagedKV.read(cache, seq, pos, dtype)
    for got, x in zip(back, (k, v)):
        if eight:
            assert torch.equal(got.double().cpu(), stored(x).to(dtype).double())
        else:
            assert torch.equal(got, x)
    # every place that no token names is as it was
    touched = torch.zeros(cache.key_pages.shape[0], page, dtype=torch.bool, device=DEV)
    touched[cache.table[seq.long(), pos.long() // page].long(), pos.long() % page] = True
    for pages in (cache.key_pages, cache.value_pages):
        rest = pages.float().transpose(1, 2)[~touched]
        assert torch.isnan(rest).all()
    if eight:
        assert (cache.key_scales.transpose(1, 2)[~touched] == 255).all()


def test_eight_bit_values_at_their_limits():
    """Zeros, the ends of the types, a vector just above and at 448 * 2^e, subnormals, infinities and NaN."""
    d, rows = 64, []

    def row(*values):
        rows.append(torch.tensor(list(values) + [0.0] * (d - len(values)), dtype=torch.float64))
    row()
    row(448.0, -448.0, 1.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10)
    row(450.0, 449.0, 1.0)
    row(3.0e38, 1.0e30)
    row(1e-40, -5e-41)
    row(2.0 ** -133)
    row(float("inf"), 5.0, -7.0)
    row(float("nan"), 0.25, float("-inf"))
    row(*[0.01 * i for i in range(d)])
    x = torch.stack(rows).to(torch.bfloat16)[:, None, :].to(DEV)
    cache = poisoned([len(rows)], 1, d, 16, torch.bfloat16, True)
    seq, pos = tokens_of([len(rows)])
    FusedPagedKV.write(cache, x, x.flip(0), seq, pos)
    key, value = FusedPagedKV.read(cache, seq, pos, torch.bfloat16)
    for got, src in ((key, x), (value, x.flip(0))):
        want = stored(src)
        # (bf16 holds every product; below its subnormals' step the multiplication rounds or flushes)
        ok = (got.double().cpu() == want) | (want.isnan() & got.isnan().cpu()) | (want.abs() < 2.0 ** -120)
        assert ok.all()
        assert (got.double().cpu() - want).nan_to_num(0.0).abs().max() <= 2.0 ** -120


def test_tokens_without_a_place_are_passed_over():
    cache = poisoned([20, 40], 2, 64, 16, torch.bfloat16, False)
    cache.table[1, 1] = 10 ** 6   # a page that the pool does not have
    cache.table[1, 2] = -1
    before = cache.key_pages.clone()
    seq = torch.tensor([0, 0, -1, 2, 1, 1, 0, 1], dtype=torch.int32, device=DEV)
    pos = torch.tensor([-1, 48, 3, 3, 17, 33, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=DEV)
    x = randn((8, 2, 64), torch.bfloat16, seed=1).to(DEV)
    FusedPagedKV.write(cache, x, x, seq, pos)
    assert torch.equal(cache.key_pages.view(torch.int16), before.view(torch.int16))
    key, value = FusedPagedKV.read(cache, seq, pos, torch.bfloat16)
    assert not key.any() and not value.any()


def test_write_reads_views_where_they_lie():
    """Slices of a packed projection, and a stride that needs a copy."""
    lengths, hkv, d = [9, 30], 2, 128
    row = randn((39, 3 * hkv * d), torch.float16, seed=6).to(DEV)
    k, v = row[:, hkv * d:2 * hkv * d].view(39, hkv, d), row[:, 2 * hkv * d:].view(39, hkv, d)
    odd = torch.empty((39, hkv, d + 1), dtype=k.dtype, device=DEV)[:, :, :d].copy_(v)
    seq, pos = tokens_of(lengths)
    for eight in (False, True):
        a, b = (poisoned(lengths, hkv, d, 16, torch.float16, eight) for _ in range(2))
        FusedPagedKV.write(a, k, odd, seq, pos)
        FusedPagedKV.write(b, k.contiguous(), v.contiguous(), seq, pos)
        for x, y in zip(FusedPagedKV.read(a, seq, pos, torch.float16), FusedPagedKV.read(b, seq, pos, torch.float16)):
            assert torch.equal(x, y)


def filled(lengths, kv_heads, d, page, dtype, eight, seed=0):
    """A poisoned cache with the positions below the lengths written."""
    cache = poisoned(lengths, kv_heads, d, page, dtype, eight, seed)
    seq, pos = tokens_of(lengths)
    k, v = (randn((len(seq), kv_heads, d), dtype, seed=seed + s).to(DEV) for s in (1, 2))
    FusedPagedKV.write(cache, k, v, seq, pos)
    key, value = FusedPagedKV.read(cache, seq, pos, dtype)
    return cache, key.split(list(lengths)), value.split(list(lengths))


def check_decode(out, q, keys, values, lengths, scale, window, dtype):
    group = q.shape[1] // keys[0].shape[1]
    for i, n in enumerate(lengths):
        if n == 0:
            assert not out[i].any()
            continue
        first = max(0, n - window) if window else 0
        for h in range(q.shape[1]):
            k, v = keys[i][first:n, h // group].double(), values[i][first:n, h // group].double()
            p = torch.softmax(k @ q[i, h].double() * scale, 0)
            want, mag = p @ v, p @ v.abs()
            bar = 1.05 * REL[dtype] * (want.abs() + mag) + 2.0 ** -15 * mag + 1e-7
            ratio = ((out[i, h].double() - want).abs() / bar).max().item()
            assert torch.isfinite(out[i, h]).all(), (i, h, n)
            assert ratio <= 1.0, f"sequence {i} of {n}, head {h}: {ratio:.2f} of the bar"


DECODE = [([1], 1, 1, 64, 16, 0), ([0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65], 2, 1, 128, 16, 0),
          ([300, 2, 128, 129, 127], 12, 12, 64, 32, 0), ([1000, 0, 257], 8, 2, 256, 64, 0),
          ([4100, 33], 7, 1, 128, 128, 0), ([700, 90, 3], 16, 1, 64, 16, 0), ([513, 260], 34, 2, 128, 16, 0),
          ([800, 100, 50, 1], 4, 4, 128, 16, 50), ([2500, 31], 6, 3, 256, 64, 1), ([900, 901, 7], 5, 5, 64, 16, 300),
          ([9000], 8, 8, 64, 16, 0)]


@pytest.mark.parametrize("dtype", HALVES, ids=IDS.get)
@pytest.mark.parametrize("eight", [False, True], ids=["16bit", "8bit"])
@pytest.mark.parametrize("lengths,heads,kv_heads,d,page,window", DECODE, ids=lambda v: str(v).replace(" ", ""))
def test_decode_attention(lengths, heads, kv_heads, d, page, window, eight, dtype):
    """Every place outside the visible positions holds NaN, pages end inside tiles."""
    cache, keys, values = filled(lengths, kv_heads, d, page, dtype, eight, seed=sum(lengths))
    q = randn((len(lengths), heads, d), dtype, seed=77).to(DEV)
    scale = 1.0 / math.sqrt(d)
    out = FusedPagedDecodeAttention.apply(q, cache, torch.tensor(lengths, dtype=torch.int32, device=DEV), scale,
                                          window or None)
    check_decode(out, q, keys, values, lengths, scale, window, dtype)
    if window:  # pages wholly before the window may have been given back
        cache.table[0, :max(0, lengths[0] - window) // page] = -1
        again = FusedPagedDecodeAttention.apply(q, cache, torch.tensor(lengths, dtype=torch.int32, device=DEV), scale,
                                                window)
        assert torch.equal(again, out)


@pytest.mark.parametrize("eight", [False, True], ids=["16bit", "8bit"])
@pytest.mark.parametrize("count,longest,window", [(64, 200, 0), (65, 300, 0), (300, 150, 40), (4097, 40, 0), (9000, 33, 5)])
def test_decode_of_many_sequences(count, longest, window, eight):
    """Numbers of sequences around those that one wave, one block and one pass of the chunks' list take."""
    heads, kv_heads, d, page, dtype = 2, 1, 64, 16, torch.bfloat16
    lengths = torch.randint(0, longest + 1, (count,), generator=torch.Generator().manual_seed(count)).tolist()
    cache, keys, values = filled(lengths, kv_heads, d, page, dtype, eight, seed=count)
    q = randn((count, heads, d), dtype, seed=7).to(DEV)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    out = FusedPagedDecodeAttention.apply(q, cache, n, 0.125, window or None)
    k, v = (torch.nn.utils.rnn.pad_sequence(x, batch_first=True)[:, :, 0].double() for x in (keys, values))
    at = torch.arange(k.shape[1], device=DEV)[None, :]
    hidden = (at >= n[:, None]) | ((at < n[:, None] - window) if window else torch.zeros_like(at, dtype=torch.bool))
    s = (q.double() @ k.transpose(1, 2) * 0.125).masked_fill(hidden[:, None], -math.inf)
    p = torch.softmax(s, -1).nan_to_num(0.0)  # (a sequence of nothing)
    want, mag = p @ v, p @ v.abs()
    assert torch.isfinite(out).all()
    assert ((out.double() - want).abs() <= 1.05 * REL[dtype] * (want.abs() + mag) + 2.0 ** -15 * mag + 1e-7).all()
    assert not out[n == 0].any()


def test_the_last_launch_of_many_sequences_is_of_the_calls_kind():
    """4096 sequences in one launch, a block each; one more, of a thousand positions, in a second."""
    lengths = torch.randint(0, 41, (4097,), generator=torch.Generator().manual_seed(1)).tolist()
    lengths[-1] = 1000
    cache, keys, values = filled(lengths, 1, 64, 1024, torch.bfloat16, False, seed=2)
    q = randn((4097, 2, 64), torch.bfloat16, seed=3).to(DEV)
    out = FusedPagedDecodeAttention.apply(q, cache, torch.tensor(lengths, dtype=torch.int32, device=DEV), 0.125)
    some = [0, 1, 2, 4094, 4095, 4096]
    check_decode(out[some], q[some], [keys[i] for i in some], [values[i] for i in some], [lengths[i] for i in some], 0.125,
                 0, torch.bfloat16)


def test_decode_scores_far_apart():
    """A maximum that keeps rising by more than an exponential can hold, and one key that outweighs the rest."""
    n, d = 500, 64
    cache, keys, values = filled([n, n], 2, d, 16, torch.bfloat16, False, seed=3)
    seq, pos = tokens_of([n, n])
    ramp = torch.arange(n, device=DEV, dtype=torch.float32)
    k = torch.stack([key.float() for key in keys])
    k[0] *= (ramp / 10)[:, None, None]
    k[1, 250] *= 100.0
    k = k.to(torch.bfloat16)
    FusedPagedKV.write(cache, k.view(2 * n, 2, d), torch.cat(values), seq, pos)
    q = randn((2, 4, d), torch.bfloat16, seed=5, std=4.0).to(DEV)
    out = FusedPagedDecodeAttention.apply(q, cache, torch.tensor([n, n], dtype=torch.int32, device=DEV), 1.0)
    # scores of several thousand: the fp32 sums behind them are off by up to 3 * 2^-24 of sum |q k| (rounding of the
    # products' partial sums), which is `slack` of an exponent and moves a probability by that much
    group = 2
    for i in range(2):
        for h in range(4):
            kk, vv = k[i, :, h // group].double(), values[i][:, h // group].double()
            s = kk @ q[i, h].double()
            p = torch.softmax(s, 0)
            slack = 3 * 2.0 ** -24 * (kk.abs() @ q[i, h].double().abs()).max()
            mag = p @ vv.abs()
            bar = 1.05 * REL[torch.bfloat16] * ((p @ vv).abs() + mag) + 2 * (slack + 2.0 ** -15) * mag + 1e-7
            assert ((out[i, h].double() - p @ vv).abs() <= bar).all()


def test_lengths_and_pages_that_the_cache_does_not_have():
    lengths = [40, 40, 40, 40]
    cache, keys, values = filled(lengths, 2, 64, 16, torch.bfloat16, False, seed=1)
    q = randn((4, 4, 64), torch.bfloat16, seed=2).to(DEV)
    given = torch.tensor([40, 49, -5, 40], dtype=torch.int32, device=DEV)  # a table of 48 positions
    cache.table[3, 1] = 10 ** 6
    out = FusedPagedDecodeAttention.apply(q, cache, given, 0.125)
    check_decode(out[:1], q[:1], keys[:1], values[:1], [40], 0.125, 0, torch.bfloat16)
    assert torch.isnan(out[1]).all() and not out[2].any() and torch.isnan(out[3]).all()
    cache.table[3, 1] = -1
    assert torch.isnan(FusedPagedDecodeAttention.apply(q, cache, given, 0.125)[3]).all()
    given[3] = 16  # (not visible then)
    assert torch.isfinite(FusedPagedDecodeAttention.apply(q, cache, given, 0.125)[3]).all()


def test_offsets_past_32_bits():
    """Places more than 2^32 bytes (and 2^31 elements) into the pool."""
    hkv, page, d = 8, 64, 128
    num_pages = 2 ** 32 // (hkv * page * d * 2) + 70     # 4.3 GiB a tensor
    pages = [torch.empty((num_pages, hkv, page, d), dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    table = torch.tensor([[num_pages - 1, 0, num_pages - 5], [3, num_pages - 2, 7]], dtype=torch.int32, device=DEV)
    cache = PagedKV(*pages, table)
    lengths = [150, 130]
    seq, pos = tokens_of(lengths)
    k, v = (randn((280, hkv, d), torch.bfloat16, seed=s).to(DEV) for s in (1, 2))
    FusedPagedKV.write(cache, k, v, seq, pos)
    back = FusedPagedKV.read(cache, seq, pos, torch.bfloat16)
    assert torch.equal(back[0], k) and torch.equal(back[1], v)
    assert torch.equal(cache.key_pages[num_pages - 1, :, 5], k[5])
    q = randn((2, 8, d), torch.bfloat16, seed=3).to(DEV)
    out = FusedPagedDecodeAttention.apply(q, cache, torch.tensor(lengths, dtype=torch.int32, device=DEV), 0.09)
    check_decode(out, q, k.split(lengths), v.split(lengths), lengths, 0.09, 0, torch.bfloat16)


def test_a_captured_step_follows_the_lengths():
    """Write and attention captured once (two graphs, each with its own workspace),
    replayed in turn while the sequences grow, between eager steps."""
    start, capacity, h, hkv, d = [5, 30, 700], 1024, 4, 2, 64
    table, total = make_table([capacity // 16] * 3)
    caches = [PagedKV.allocate(table.to(DEV), total, hkv, 16, d, torch.bfloat16, DEV, quantized=True) for _ in range(3)]
    seq, pos = tokens_of(start)
    for c in caches:
        FusedPagedKV.write(c, *(randn((sum(start), hkv, d), torch.bfloat16, seed=s).to(DEV) for s in (1, 2)), seq, pos)
    rows = torch.arange(3, dtype=torch.int32, device=DEV)
    q, k, v = torch.empty((3, h, d), dtype=torch.bfloat16, device=DEV), *(
        torch.empty((3, hkv, d), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    lengths = torch.tensor(start, dtype=torch.int32, device=DEV)

    def step(cache):
        FusedPagedKV.write(cache, k, v, rows, lengths)
        return FusedPagedDecodeAttention.apply(q, cache, lengths + 1, 0.125)
    graphs = []
    for cache in caches[:2]:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(cache)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(cache)
        graphs.append((graph, out))
    for i in range(40):
        for x, s in ((q, 10), (k, 20), (v, 30)):
            x.copy_(randn(x.shape, x.dtype, seed=100 * i + s))
        for graph, _ in graphs:
            graph.replay()
        want = step(caches[2])
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want), i
        lengths += 1


def test_two_streams_at_once():
    lengths = [5000, 1200, 3]
    cache, keys, values = filled(lengths, 4, 128, 64, torch.bfloat16, False, seed=9)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    qs = [randn((3, 16, 128), torch.bfloat16, seed=s).to(DEV) for s in (1, 2)]
    want = [FusedPagedDecodeAttention.apply(q, cache, n, 0.09) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(FusedPagedDecodeAttention.apply(qs[i], cache, n, 0.09))
    torch.cuda.synchronize()
    for w, got in zip(want, outs):
        assert all(torch.equal(w, x) for x in got)


def test_refused_calls():
    cache, _, _ = filled([20, 30], 2, 64, 16, torch.bfloat16, False)
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device=DEV)
    n = torch.tensor([20, 30], dtype=torch.int32, device=DEV)
    x = torch.zeros((2, 2, 64), dtype=torch.bfloat16, device=DEV)
    for bad in (lambda: FusedPagedDecodeAttention.apply(q.half(), cache, n, 1.0),
                lambda: FusedPagedDecodeAttention.apply(q[:1], cache, n[:1], 1.0),
                lambda: FusedPagedDecodeAttention.apply(q[:, :3], cache, n, 1.0),
                lambda: FusedPagedDecodeAttention.apply(q[:, :, :32], cache, n, 1.0),
                lambda: FusedPagedDecodeAttention.apply(q, cache, n.long(), 1.0),
                lambda: FusedPagedDecodeAttention.apply(q, cache, n.cpu(), 1.0),
                lambda: FusedPagedDecodeAttention.apply(q, cache, n, 0.0),
                lambda: FusedPagedDecodeAttention.apply(q.clone().requires_grad_(True), cache, n, 1.0),
                lambda: FusedPagedKV.write(cache, x, x.half(), n, n),
                lambda: FusedPagedKV.write(cache, x.half(), x.half(), n, n),
                lambda: FusedPagedKV.write(cache, x, x, n[:1], n),
                lambda: FusedPagedKV.write(cache, x[:, :1], x[:, :1], n, n),
                lambda: FusedPagedKV.write(cache, x.clone().requires_grad_(True), x, n, n),
                lambda: FusedPagedKV.read(cache, n, n, torch.float32),
                lambda: FusedPagedKV.read(cache, n, n, torch.float16)):
        with pytest.raises(RuntimeError):
            bad()
    assert FusedPagedDecodeAttention.is_available(q, cache)
    assert not FusedPagedDecodeAttention.is_available(q.half(), cache)
    assert not FusedPagedDecodeAttention.is_available(q, cache, True, 0.1)


def test_eight_bit_values_at_the_ends_of_fp16():
    """Every finite fp16 number comes back finite: at the top the nearest number of the storage that fp16 has, 240 * 2^8;
    below the normal numbers the product rounded to fp16."""
    d, rows = 64, []

    def row(*values):
        rows.append(torch.tensor(list(values) + [0.0] * (d - len(values)), dtype=torch.float64))
    row(65504.0, -65504.0, 63520.0, 63488.0, 63456.0, -61472.0, 61440.0, 59000.0, 1.0, 0.25)
    row(-61472.0, 3.0)
    row(57376.0, 100.0)
    row(57344.0, -57344.0, 100.0)
    row(60000.0, float("inf"), float("nan"), -65504.0)
    row(2.0 ** -24, -2.0 ** -23, 3 * 2.0 ** -24)
    row(2.0 ** -14, 2.0 ** -15, 2.0 ** -24, 1023 * 2.0 ** -24)
    x = torch.stack(rows).to(torch.float16)[:, None, :].to(DEV)
    assert x[0, 0, 0] == 65504.0
    cache = poisoned([len(rows)], 1, d, 16, torch.float16, True)
    seq, pos = tokens_of([len(rows)])
    FusedPagedKV.write(cache, x, x.flip(0), seq, pos)
    key, value = FusedPagedKV.read(cache, seq, pos, torch.float16)
    for got, src in ((key, x), (value, x.flip(0))):
        want = stored(src.clamp(-61440.0, 61440.0).where(src.isfinite(), src)).to(torch.float16)
        assert torch.equal(got.cpu().nan_to_num(7.0), want.nan_to_num(7.0)) and torch.equal(got.isnan().cpu(), want.isnan())
        assert torch.equal(got.isfinite(), src.isfinite())


@pytest.mark.parametrize("d", [64, 128, 256])
def test_large_values_of_keys_that_do_not_count(d):
    """A value at the end of fp16 under a probability that rounds to zero changes nothing."""
    n, dtype = 70, torch.float16
    cache = poisoned([n], 2, d, 16, dtype, True)
    seq, pos = tokens_of([n])
    k, v = (randn((n, 2, d), dtype, seed=s).to(DEV) for s in (1, 2))
    q = randn((1, 4, d), dtype, seed=3).to(DEV)
    q[..., 0] = 1.0
    k[..., 0] = 0.0
    k[33, :, 0] = -1000.0
    v[33, :, :] = 65504.0
    v[33, :, 1::2] = -65504.0
    FusedPagedKV.write(cache, k, v, seq, pos)
    key, value = FusedPagedKV.read(cache, seq, pos, dtype)
    assert value.isfinite().all()
    out = FusedPagedDecodeAttention.apply(q, cache, torch.tensor([n], dtype=torch.int32, device=DEV), 0.125)
    check_decode(out, q, [key], [value], [n], 0.125, 0, dtype)
    assert out.abs().max() < 10.0


@pytest.mark.parametrize("n,heads,kv_heads,d", [(70, 4, 2, 64), (300, 2, 2, 128), (900, 16, 1, 256), (6000, 4, 4, 64)],
                         ids=lambda v: str(v))
def test_keys_with_infinite_scores_count_as_nothing(n, heads, kv_heads, d):
    """Scores of -inf, over whole tiles and chunks, at the start, in the middle and at the end, beside ordinary ones;
    only such scores: NaN, as the formula gives."""
    dtype = torch.bfloat16
    cache = poisoned([n, n], kv_heads, d, 64, dtype, False)
    seq, pos = tokens_of([n, n])
    k, v = (randn((2 * n, kv_heads, d), dtype, seed=s).to(DEV) for s in (1, 2))
    q = randn((2, heads, d), dtype, seed=3).to(DEV)
    q[..., 0] = 1.0
    at = torch.arange(n, device=DEV)
    gone = (at < n // 3) | ((at > n // 2) & (at < n // 2 + 5)) | (at >= n - 40)
    k[:n][gone, :, 0] = -math.inf
    k[n:, :, 0] = -math.inf
    FusedPagedKV.write(cache, k, v, seq, pos)
    out = FusedPagedDecodeAttention.apply(q, cache, torch.tensor([n, n], dtype=torch.int32, device=DEV), 0.1)
    check_decode(out[:1], q[:1], [k[:n]], [v[:n]], [n], 0.1, 0, dtype)
    assert out[1].isnan().all()
    rest = FusedPagedDecodeAttention.apply(q, cache, torch.tensor([n // 3 + 1, n], dtype=torch.int32, device=DEV), 0.1, 1)
    assert torch.equal(rest[0], v[n // 3].repeat_interleave(heads // kv_heads, 0))
