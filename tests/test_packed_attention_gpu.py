"""Attention over packed sequences, forward and gradients, against the formulas
in float64 on the device.

Tolerance. With REL half a step of the storage type (2^-8 bf16, 2^-11 fp16):
  * out is an fp32 sum of rounded probabilities times v, rounded once:
        REL * (P |v|) + REL * |out|
  * the gradients' bounds are those of the dense backward: each is an fp32 sum
    rounded once (REL * |ref|); P and dS are rounded before the products that
    sum them (REL * P^T |dO|, REL * scale * |dS| |K|, REL * scale * |dS|^T |Q|);
    delta comes from an output with the probabilities' rounding in it (dS off by
    scale * P * REL * sum |dO| (P |v|)).
  * scores are fp32 sums of up to 256 products and an exponential of one step:
    below 2^-15 of every probability.
The bar is 1.05 times the sum for the output, twice the sum for the gradients
(both roundings of P and dS meet in them), each with 2^-15 of the summed
magnitudes added."""

import ctypes
import math

import pytest
import torch

from oslo_amd import FusedPackedAttention, FusedPrefillAttention, PackedSequences, _lib, kernels
from tests.util import IDS, randn

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
REL = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
HALVES = [torch.float16, torch.bfloat16]
FP32 = 2.0 ** -15


def make(lengths, heads, kv_heads, d, dtype, seed, tail=0):
    t = sum(lengths) + tail
    q = randn((t, heads, d), dtype, seed).to(DEV)
    k, v = (randn((t, kv_heads, d), dtype, seed + i).to(DEV) for i in (1, 2))
    g = randn((t, heads, d), dtype, seed + 3).to(DEV)
    return q, k, v, g


def reference(q, k, v, g, lengths, scale, window=0):
    """float64 (out, dq, dk, dv) and the bounds' sums, over [T, heads, D]."""
    heads, kv_heads = q.shape[1], k.shape[1]
    group = heads // kv_heads
    out = [torch.zeros(x.shape, dtype=torch.float64, device=q.device) for x in (q, q, k, v)]
    mag = [torch.zeros_like(x) for x in out]
    start = 0
    for n in lengths:
        rows = slice(start, start + n)
        start += n
        i = torch.arange(n, device=q.device)
        hidden = i[None, :] > i[:, None]
        if window:
            hidden = hidden | (i[None, :] <= i[:, None] - window)
        for h in range(heads):
            qs, ks, vs, gs = (x[rows, c].double() for x, c in ((q, h), (k, h // group), (v, h // group), (g, h)))
            p = torch.softmax((qs @ ks.t() * scale).masked_fill(hidden, -math.inf), -1)
            o = p @ vs
            dp = gs @ vs.t()
            ds = p * (dp - (gs * o).sum(-1, keepdim=True))
            # what moves dS: its own rounding, and delta's, which comes from rounded probabilities
            ds_mag = ds.abs() + p * (gs.abs() * (p @ vs.abs())).sum(-1, keepdim=True)
            out[0][rows, h], out[1][rows, h] = o, scale * (ds @ ks)
            out[2][rows, h // group] += scale * (ds.t() @ qs)
            out[3][rows, h // group] += p.t() @ gs
            mag[0][rows, h] = p @ vs.abs()
            mag[1][rows, h] = scale * (ds_mag @ ks.abs())
            mag[2][rows, h // group] += scale * (ds_mag.t() @ qs.abs())
            mag[3][rows, h // group] += p.t() @ gs.abs()
    return out, mag


def check(got, want, mag, dtype, factor, what):
    bar = factor * REL[dtype] * (want.abs() + mag) + FP32 * mag + 1e-7
    ratio = ((got.double() - want).abs() / bar).max().item() if want.numel() else 0.0
    assert torch.isfinite(got).all(), what
    assert ratio <= 1.0, f"{what}: {ratio:.2f} of the bar"


CASES = [([1], 2, 2, 64, 0), ([1, 1, 1], 4, 2, 128, 0), ([0, 5, 0, 128, 129, 127, 0], 6, 1, 64, 0),
         ([300, 31, 33, 64], 7, 7, 128, 0), ([513, 2], 4, 2, 256, 0), ([200, 17], 6, 3, 256, 17),
         ([400, 130, 1], 8, 2, 128, 1), ([700, 65], 5, 5, 64, 256), ([1100], 12, 12, 64, 300), ([260, 260], 16, 2, 128, 259)]


# one long sequence, few key/value heads: the longest dK/dV walks are shared over a group's heads
SHARED = [([2000], 8, 1, 128, 0), ([1500, 3], 16, 2, 256, 0), ([1700, 200], 12, 1, 64, 0), ([2100], 8, 2, 128, 1500)]


@pytest.mark.parametrize("dtype", HALVES, ids=IDS.get)
@pytest.mark.parametrize("lengths,heads,kv_heads,d,window", SHARED, ids=lambda v: str(v).replace(" ", ""))
def test_gradients_of_shared_walks(lengths, heads, kv_heads, d, window, dtype):
    split, parts = PackedSequences(lengths, "cpu").shared_blocks(heads, kv_heads, d, window)
    assert split > 0 and parts > 1
    test_output_and_gradients(lengths, heads, kv_heads, d, window, dtype)


@pytest.mark.parametrize("dtype", HALVES, ids=IDS.get)
@pytest.mark.parametrize("lengths,heads,kv_heads,d,window", CASES, ids=lambda v: str(v).replace(" ", ""))
def test_output_and_gradients(lengths, heads, kv_heads, d, window, dtype):
    q, k, v, g = make(lengths, heads, kv_heads, d, dtype, seed=sum(lengths) + d, tail=3)
    packed = PackedSequences(lengths, DEV)
    scale = 1.0 / math.sqrt(d)
    want, mag = reference(q, k, v, g, lengths, scale, window)
    out = FusedPackedAttention.apply(q, k, v, packed, scale, window or None)
    check(out, want[0], mag[0], dtype, 1.05, "out")
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    trained = FusedPackedAttention.apply(*leaves, packed, scale, window or None)
    assert torch.equal(trained, out)
    grads = torch.autograd.grad(trained, leaves, g)
    for name, got, w, m in zip(("dq", "dk", "dv"), grads, want[1:], mag[1:]):
        check(got, w, m, dtype, 2.0, name)
        assert not got[packed.total:].any()
    assert not out[packed.total:].any()


def test_gradients_against_differences():
    """The directional derivative of sum(g * out) in float64, by differences, against
    the kernel's gradients along the same direction."""
    lengths, scale, dtype = [70, 200, 3], 0.125, torch.bfloat16
    q, k, v, g = make(lengths, 4, 2, 64, dtype, seed=5)
    packed = PackedSequences(lengths, DEV)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    grads = torch.autograd.grad(FusedPackedAttention.apply(*leaves, packed, scale), leaves, g)
    want, mag = reference(q, k, v, g, lengths, scale)
    step = 1e-4
    for i, name in enumerate("qkv"):
        direction = randn(leaves[i].shape, torch.float32, seed=30 + i).to(DEV).double()
        values = []
        for sign in (1, -1):
            moved = [x.double() for x in (q, k, v)]
            moved[i] = moved[i] + sign * step * direction
            values.append((reference(*moved, g.double(), lengths, scale)[0][0] * g.double()).sum())
        slope = (values[0] - values[1]) / (2 * step)
        bar = ((2 * REL[dtype] * (want[1 + i].abs() + mag[1 + i]) + FP32 * mag[1 + i]) * direction.abs()).sum()
        assert abs((grads[i].double() * direction).sum() - slope) <= bar + 1e-3 * slope.abs(), name


@pytest.mark.parametrize("dtype", HALVES, ids=IDS.get)
def test_equals_the_prompt_attention(dtype):
    """Equal lengths and heads: the packed kernel does the arithmetic of the dense one (but for the row sums
    of the gradients of queries and keys, which it takes from the output before its rounding)."""
    b, h, s, d = 3, 4, 260, 128
    q, k, v, g = make([s] * b, h, h, d, dtype, seed=9)
    packed = PackedSequences([s] * b, DEV)
    dense = [x.view(b, s, h, d).permute(0, 2, 1, 3).detach().requires_grad_(True) for x in (q, k, v)]
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    out = FusedPackedAttention.apply(*leaves, packed, 0.1)
    ref = FusedPrefillAttention.apply(*dense, None, 0.1)
    assert torch.equal(out.view(b, s, h, d).permute(0, 2, 1, 3), ref)
    got = torch.autograd.grad(out, leaves, g)
    want = torch.autograd.grad(ref, dense, g.view(b, s, h, d).permute(0, 2, 1, 3))
    assert torch.equal(got[2].view(b, s, h, d).permute(0, 2, 1, 3), want[2])


def test_sequences_do_not_see_each_other():
    """NaN and infinities in one sequence, and in the rows behind the last, stay there."""
    lengths = [40, 150, 33]
    q, k, v, g = make(lengths, 4, 2, 64, torch.bfloat16, seed=21, tail=5)
    packed = PackedSequences(lengths, DEV)

    def run(*tensors):
        leaves = [x.clone().requires_grad_(True) for x in tensors[:3]]
        out = FusedPackedAttention.apply(*leaves, packed, 0.125)
        return [out.detach()] + list(torch.autograd.grad(out, leaves, tensors[3]))
    clean = run(q, k, v, g)
    spoilt = [x.clone() for x in (q, k, v, g)]
    for x in spoilt:
        x[40:190] = float("nan")
        x[45] = float("inf")
        x[223:] = float("nan")
    for x, y in zip(run(*spoilt), clean):
        assert torch.equal(x[:40], y[:40]) and torch.equal(x[190:223], y[190:223])
        assert not x[223:].any()


def test_views_are_read_where_they_lie():
    """Slices of a packed projection, an odd stride (copied) and an expanded gradient."""
    lengths, h, hkv, d = [90, 40], 4, 2, 64
    row = randn((130, (h + 2 * hkv) * d), torch.float16, seed=3).to(DEV)
    q = row[:, :h * d].view(130, h, d)
    k = row[:, h * d:(h + hkv) * d].view(130, hkv, d)
    v = row[:, (h + hkv) * d:].view(130, hkv, d)
    packed = PackedSequences(lengths, DEV)
    want = FusedPackedAttention.apply(q.contiguous(), k.contiguous(), v.contiguous(), packed, 0.125)
    assert torch.equal(FusedPackedAttention.apply(q, k, v, packed, 0.125), want)
    odd = torch.empty((130, h, d + 3), dtype=q.dtype, device=DEV)[:, :, :d].copy_(q)
    assert torch.equal(FusedPackedAttention.apply(odd, k, v, packed, 0.125), want)
    shared = k[:1].expand(130, hkv, d)  # a broadcast key: its gradient is the sum over the tokens
    leaf = k[:1].clone().requires_grad_(True)
    out = FusedPackedAttention.apply(q, leaf.expand(130, hkv, d), v, packed, 0.125)
    assert torch.equal(out, FusedPackedAttention.apply(q, shared.contiguous(), v, packed, 0.125))
    out.float().sum().backward()  # (an expanded gradient of ones)
    assert leaf.grad.shape == leaf.shape and torch.isfinite(leaf.grad).all()


def test_same_bits_on_every_run_and_stream():
    lengths = [700, 1, 333]
    q, k, v, g = make(lengths, 8, 2, 128, torch.bfloat16, seed=12)
    packed = PackedSequences(lengths, DEV)

    def run():
        leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
        out = FusedPackedAttention.apply(*leaves, packed, 0.09)
        return [out.detach()] + list(torch.autograd.grad(out, leaves, g))
    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    second = run()
    torch.cuda.synchronize()
    for a, b, c in zip(first, second, other):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_captured_into_a_graph():
    """Forward and gradients of a training step's attention, replayed with new
    inputs between eager calls."""
    lengths = [200, 64, 5]
    q, k, v, g = make(lengths, 4, 4, 128, torch.bfloat16, seed=40)
    packed = PackedSequences(lengths, DEV)
    static = [x.clone().requires_grad_(True) for x in (q, k, v)]
    static_g = g.clone()

    def run(leaves, grad):
        out = FusedPackedAttention.apply(*leaves, packed, 0.1, 100)
        return [out] + list(torch.autograd.grad(out, leaves, grad))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            run(static, static_g)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = run(static, static_g)
    for seed in (50, 60, 70):
        fresh = make(lengths, 4, 4, 128, torch.bfloat16, seed=seed)
        with torch.no_grad():
            for x, y in zip(static + [static_g], fresh):
                x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        want = run([x.clone().requires_grad_(True) for x in fresh[:3]], fresh[3])
        for x, y in zip(results, want):
            assert torch.equal(x.detach(), y.detach())


def test_empty_and_refused_calls():
    q = torch.zeros((5, 2, 64), dtype=torch.bfloat16, device=DEV)
    assert not FusedPackedAttention.apply(q, q, q, PackedSequences([], DEV), 0.1).any()
    assert not FusedPackedAttention.apply(q, q, q, PackedSequences([0, 0], DEV), 0.1).any()
    assert FusedPackedAttention.apply(q[:0], q[:0], q[:0], PackedSequences([0], DEV), 0.1).shape == (0, 2, 64)
    leaf = q.clone().requires_grad_(True)
    FusedPackedAttention.apply(leaf, q, q, PackedSequences([], DEV), 0.1).sum().backward()
    assert not leaf.grad.any()
    four = PackedSequences([4], DEV)
    for bad in (lambda: FusedPackedAttention.apply(q, q, q, PackedSequences([6], DEV), 0.1),
                lambda: FusedPackedAttention.apply(q.float(), q.float(), q.float(), four, 0.1),
                lambda: FusedPackedAttention.apply(q, q[:, :, :32], q[:, :, :32], four, 0.1),
                lambda: FusedPackedAttention.apply(q[:, :, :32], q[:, :, :32], q[:, :, :32], four, 0.1),
                lambda: FusedPackedAttention.apply(q, q.half(), q.half(), four, 0.1),
                lambda: FusedPackedAttention.apply(q, q[:4], q[:4], four, 0.1),
                lambda: FusedPackedAttention.apply(q[:, :1], q, q, four, 0.1),
                lambda: FusedPackedAttention.apply(q, q, q, four, -1.0),
                lambda: FusedPackedAttention.apply(q, q, q, PackedSequences([4], "cpu"), 0.1)):
        with pytest.raises(RuntimeError):
            bad()
    assert FusedPackedAttention.is_available(q, q) and not FusedPackedAttention.is_available(q, q, True, 0.1)
    assert not FusedPackedAttention.is_available(q.float(), q.float())


def test_list_entries_out_of_range_are_passed_over():
    """Entries of a hand-made list that leave the row are not followed (the kernel's own check)."""
    q, k, v, _ = make([20], 2, 2, 64, torch.bfloat16, seed=8, tail=10)
    packed = PackedSequences([20], DEV)
    want = kernels.attention_packed_forward(q, k, v, packed, 0.1)
    packed.blocks = torch.tensor([[[0, 20, 0, 0], [-1, 4, 0, 0], [25, 6, 0, 0], [0, 20, 1, 0], [0, 0, 0, 0],
                                   [0, 21, 0, 0], [3, 4, -1, 0]]] * 2, dtype=torch.int32, device=DEV)
    assert torch.equal(kernels.attention_packed_forward(q, k, v, packed, 0.1), want)


def test_a_capture_is_refused_while_an_eager_graph_of_the_same_leaf_lives():
    packed = PackedSequences([40], DEV)
    q, k, v = (torch.randn(40, 2, 64, device=DEV, dtype=torch.float16, requires_grad=True) for _ in range(3))
    grad = torch.ones(40, 2, 64, device=DEV, dtype=torch.float16)
    living = FusedPackedAttention.apply(q, k, v, packed)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(graph):
            FusedPackedAttention.apply(q, k, v, packed)
    torch.autograd.backward(living, grad)
    want = [t.grad.clone() for t in (q, k, v)]
    del living
    for t in (q, k, v):
        t.grad = None
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = FusedPackedAttention.apply(q, k, v, packed)
        torch.autograd.backward(out, grad)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for t, w in zip((q, k, v), want):
            assert torch.equal(t.grad, w)
            t.grad.zero_()


def test_tangents_of_forward_mode_are_refused():
    """The operator has no formula for them: a result without its tangent would be a wrong derivative of zero."""
    from torch.autograd import forward_ad
    q, k, v, g = make([20, 7], 4, 2, 64, torch.bfloat16, seed=14)
    packed = PackedSequences([20, 7], DEV)
    want = FusedPackedAttention.apply(q, k, v, packed, 0.1)
    with forward_ad.dual_level():
        for i in range(3):
            given = [forward_ad.make_dual(x, torch.ones_like(x)) if j == i else x for j, x in enumerate((q, k, v))]
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(RuntimeError, match="forward mode"):
                    FusedPackedAttention.apply(*given, packed, 0.1)
        assert torch.equal(FusedPackedAttention.apply(q, k, v, packed, 0.1), want)


@pytest.mark.parametrize("dtype", HALVES, ids=IDS.get)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_what_the_outputs_rounding_left_out_counts(d, dtype):
    """delta = sum dO O stands against dP in every dS of a row. Where a query sees two keys, O's own rounding is as
    large an error in it as the others together (those of P and dS before their products, and of the gradients): the
    formulas in 64 bits with each of these roundings applied are off by 0.0024 of dQ's and dK's norms in bf16, and by
    0.0037 with delta from the rounded O, 1.5 times as much, at every head size and in either type. Asked for: 1.25."""
    lengths, heads, window, scale = [260, 1, 100], 3, 2, 1.0 / math.sqrt(d)
    q, k, v, g = make(lengths, heads, heads, d, dtype, seed=d)
    packed = PackedSequences(lengths, DEV)
    want, _ = reference(q, k, v, g, lengths, scale, window)
    out, low, lse = kernels.attention_packed_forward(q, k, v, packed, scale, window, want_lse=True)
    exact = out.double() + low.double()
    assert (exact - want[0]).norm() < (out.double() - want[0]).norm()
    with_low = kernels.attention_packed_backward(g, q, k, v, out, low, lse, packed, scale, window)
    zeros = kernels.attention_packed_backward(g, q, k, v, out, torch.zeros_like(low), lse, packed, scale, window)
    # the same through the library's own argument: no tensor
    none = [torch.empty_like(x) for x in (q, k, v)]
    t, blocks = q.shape[0], packed.blocks
    lib = _lib.load()
    size = lib.oslo_attention_packed_bwd_workspace_bytes(t, heads, heads, d, 0, 1)
    workspace = torch.empty(size // 4, dtype=torch.float32, device=DEV)
    strides = (ctypes.c_int64 * 16)(*([d, heads * d] * 8))
    _lib.check(lib.oslo_attention_packed_bwd(
        *(x.data_ptr() for x in none), g.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), None,
        lse.data_ptr(), workspace.data_ptr(), blocks[0].data_ptr(), blocks[1].data_ptr(), blocks.shape[1], 0, 1, scale, t,
        packed.max_length, heads, heads, d, window, strides, 1 if dtype == torch.float16 else 2,
        torch.cuda.current_stream().cuda_stream))
    for x, y in zip(none, zeros):
        assert torch.equal(x, y)
    for i, name in ((0, "dq"), (1, "dk")):
        errors = [float((x[i].double() - want[1 + i]).norm()) for x in (with_low, zeros)]
        assert errors[1] >= 1.25 * errors[0], (name, [e / float(want[1 + i].norm()) for e in errors])
    assert torch.equal(with_low[2], zeros[2])


def test_a_capture_is_refused_while_an_eager_graph_of_the_views_leaf_lives():
    packed = PackedSequences([40], DEV)
    leaf = torch.randn(40, 3, 2, 64, device=DEV, dtype=torch.float16, requires_grad=True)
    grad = torch.ones(40, 2, 64, device=DEV, dtype=torch.float16)
    living = FusedPackedAttention.apply(*leaf.unbind(1), packed)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(graph):
            FusedPackedAttention.apply(*leaf.unbind(1), packed)
    torch.autograd.backward(living, grad)
    want = leaf.grad.clone()
    del living
    leaf.grad = None
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = FusedPackedAttention.apply(*leaf.unbind(1), packed)
        torch.autograd.backward(out, grad)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(leaf.grad, want)
        leaf.grad.zero_()


@pytest.mark.parametrize("window", [0, 150])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_keys_with_infinite_scores_count_as_nothing(d, window):
    """Scores of -inf over whole tiles at a sequence's start and later, beside ordinary ones; a query that sees no other:
    NaN, as the formula gives."""
    lengths, dtype, scale = [300, 5, 170], torch.bfloat16, 0.1
    q, k, v, _ = make(lengths, 4, 2, d, dtype, seed=d + window)
    packed = PackedSequences(lengths, DEV)
    q[..., 0] = 1.0
    at = torch.cat([torch.arange(n, device=DEV) for n in lengths])
    gone = (at < 70) | ((at > 100) & (at < 103)) | ((at > 128) & (at < 200))
    gone[300:305] = False
    k[gone, :, 0] = -math.inf
    out = FusedPackedAttention.apply(q, k, v, packed, scale, window or None)
    trained = FusedPackedAttention.apply(q.clone().requires_grad_(True), k, v, packed, scale, window or None)
    want, mag = reference(q, k, v, torch.zeros_like(q), lengths, scale, window)
    sees = ~want[0].isnan().any(-1).any(-1)
    assert sees.sum() == 475 - 140 and out[~sees].isnan().all()
    check(out[sees], want[0][sees], mag[0][sees], dtype, 1.05, "out")
    assert torch.equal(trained[sees], out[sees])
