"""The operators for batches of sequences of different lengths, as workloads:
attention over packed sequences (and its gradients), the paged key/value cache
(written in 16 or 8 bits, read back), attention of one new token per sequence
over that cache, and sampling. ``listed()`` names the cases, ``draw(rng)`` makes
more of the same ranges, ``prepare`` makes a case's inputs, ``run`` is one pass:
in elementary torch operations, or (``own``) through this package's operators.
``exact`` is the same result in 64 bits, by another route."""

import math
import random

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}
_E4M3_MAX = 448.0


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # Scoring a handful of short prompts at once with a 12-head model: a call whose latency counts.
        dict(name="packed_short", op="packed", grad=False, dtype="fp16", heads=12, kv_heads=12, head_dim=64,
             sequences=5, shortest=1, longest=61, window=0),
        # The prompts of a batch of requests, heads of 256 features: the long forward of a serving step.
        dict(name="packed_prompts", op="packed", grad=False, dtype="bf16", heads=16, kv_heads=16, head_dim=256,
             sequences=9, shortest=200, longest=2048, window=0),
        # A training step's attention: documents packed into one row, four query heads to a key/value head.
        dict(name="packed_train_grouped", op="packed", grad=True, dtype="bf16", heads=32, kv_heads=8, head_dim=128,
             sequences=7, shortest=300, longest=4095, window=0),
        # The same for a model's sliding-window layers (20 heads, 256 keys back).
        dict(name="packed_train_window", op="packed", grad=True, dtype="fp16", heads=20, kv_heads=20, head_dim=128,
             sequences=11, shortest=65, longest=2048, window=256),
        # A decoding step's new keys and values joining a 16-bit cache: one token per sequence.
        dict(name="cache_step", op="cache", dtype="bf16", stored="bf16", kv_heads=16, head_dim=256, page=32,
             sequences=64, shortest=1, longest=2047, step=True),
        # A batch of prompts written into an 8-bit cache and read back for the next part of the prompt.
        dict(name="cache_prompts_8bit", op="cache", dtype="bf16", stored="e4m3", kv_heads=16, head_dim=256, page=64,
             sequences=24, shortest=77, longest=2048, step=False),
        # One long conversation, grouped heads: a single row of work that has to be split to fill the card.
        dict(name="decode_one_long", op="decode", dtype="bf16", stored="bf16", heads=32, kv_heads=8, head_dim=128,
             page=64, sequences=1, shortest=131071, longest=131071, window=0),
        # A few short conversations with a 12-head model: latency.
        dict(name="decode_short", op="decode", dtype="fp16", stored="fp16", heads=12, kv_heads=12, head_dim=64,
             page=16, sequences=4, shortest=1, longest=300, window=0),
        # A full serving batch over an 8-bit cache with grouped heads, lengths spread widely.
        dict(name="decode_batch_8bit", op="decode", dtype="bf16", stored="e4m3", heads=32, kv_heads=8, head_dim=128,
             page=64, sequences=128, shortest=100, longest=8191, window=0),
        # One sequence, the usual mixture of filters: latency.
        dict(name="sample_one", op="sample", dtype="fp32", rows=1, vocab=50257, per_row=False, temperature=0.8,
             top_k=50, top_p=0.95, min_p=0.0, banned=3),
        # A serving batch in which every request brings settings of its own.
        dict(name="sample_batch", op="sample", dtype="bf16", rows=256, vocab=50400, per_row=True, temperature=1.0,
             top_k=0, top_p=0.9, min_p=0.05, banned=8),
        # Many rows at once (several samples per prompt, scoring), nucleus sampling over the whole vocabulary.
        dict(name="sample_many", op="sample", dtype="fp32", rows=1000, vocab=50257, per_row=False, temperature=1.0,
             top_k=0, top_p=0.92, min_p=0.0, banned=0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    limits = [work(case) for case in listed()]
    while True:  # (no drawn case moves or computes more than the largest listed one)
        case = _draw(rng)
        cost = work(case)
        if all(cost[what] <= max(w[what] for w in limits) for what in ("bytes", "flops")):
            return case


def _draw(rng):
    kind = rng.choice(["packed", "packed", "cache", "decode", "decode", "sample"])
    if kind == "sample":
        return dict(op="sample", dtype=rng.choice(["fp32", "bf16", "fp16"]), rows=_log_int(rng, 1, 1000),
                    vocab=_log_int(rng, 40, 70000), per_row=rng.random() < 0.5,
                    temperature=round(rng.uniform(0.3, 1.6), 3), top_k=rng.choice([0, 0, 1, 20, _log_int(rng, 2, 5000)]),
                    top_p=rng.choice([1.0, round(rng.uniform(0.05, 0.99), 3)]),
                    min_p=rng.choice([0.0, round(rng.uniform(0.001, 0.3), 4)]), banned=rng.choice([0, 5]))
    head_dim = rng.choice([64, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 5, 8, 12, 16])
    heads = kv_heads * rng.choice([1, 1, 2, 4, 7] if kv_heads <= 8 else [1])
    dtype = rng.choice(["bf16", "fp16"])
    window = rng.choice([0, 0, 0, 256, _log_int(rng, 1, 1500)])
    if kind == "packed":
        longest = _log_int(rng, 1, 3000)
        sequences = rng.randint(1, max(1, min(40, 9000 // longest)))
        return dict(op="packed", grad=rng.random() < 0.5, dtype=dtype, heads=heads, kv_heads=kv_heads,
                    head_dim=head_dim, sequences=sequences, shortest=_log_int(rng, 1, longest), longest=longest,
                    window=window)
    page = rng.choice([16, 32, 64, 128])
    stored = rng.choice([dtype, "e4m3"])
    if kind == "cache":
        longest = _log_int(rng, 1, 4000)
        sequences = rng.randint(1, max(1, min(100, 20000 // longest)))
        return dict(op="cache", dtype=dtype, stored=stored, kv_heads=kv_heads, head_dim=head_dim, page=page,
                    sequences=sequences, shortest=_log_int(rng, 1, longest), longest=longest, step=rng.random() < 0.3)
    longest = _log_int(rng, 1, 60000)
    sequences = rng.randint(1, max(1, min(150, 200000 // longest)))
    return dict(op="decode", dtype=dtype, stored=stored, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page,
                sequences=sequences, shortest=_log_int(rng, 1, longest), longest=longest, window=window)


def _lengths(case):
    """The sequences' lengths: spread over their logarithm, the longest among them."""
    rng = random.Random(case["sequences"] * 1000003 + case["longest"])
    out = [_log_int(rng, case["shortest"], case["longest"]) for _ in range(case["sequences"])]
    out[rng.randrange(len(out))] = case["longest"]
    return out


def _pairs(length, window):
    """Visible (query, key) pairs of one sequence."""
    if window <= 0 or window >= length:
        return length * (length + 1) // 2
    return window * (window + 1) // 2 + (length - window) * window


def work(case):
    if case["op"] == "packed":
        lengths, d = _lengths(case), case["head_dim"]
        tokens = sum(lengths)
        pairs = sum(_pairs(n, case["window"]) for n in lengths)
        q, kv = tokens * case["heads"] * d * 2, tokens * case["kv_heads"] * d * 2
        # forward: q, k, v in, out; with gradients also the output's gradient in and three gradients out
        moved = 2 * q + 2 * kv + ((2 * q + 2 * kv) if case["grad"] else 0)
        return {"bytes": moved, "flops": (14 if case["grad"] else 4) * d * case["heads"] * pairs}
    if case["op"] == "cache":
        tokens = case["sequences"] if case["step"] else sum(_lengths(case))
        rows = 2 * tokens * case["kv_heads"]
        d, stored = case["head_dim"], _BYTES[case["stored"]]
        scales = 1 if case["stored"] == "e4m3" else 0
        moved = rows * (d * 2 + d * stored + scales)  # the write
        if case["stored"] == "e4m3":
            moved += rows * (d * stored + scales + d * 2)  # and the reading back
        return {"bytes": moved, "flops": rows * d * (3 if case["stored"] == "e4m3" else 0)}
    if case["op"] == "decode":
        visible = sum(min(n, case["window"]) if case["window"] else n for n in _lengths(case))
        d, stored = case["head_dim"], _BYTES[case["stored"]]
        scales = 1 if case["stored"] == "e4m3" else 0
        return {"bytes": 2 * visible * case["kv_heads"] * (d * stored + scales)
                + 2 * case["sequences"] * case["heads"] * d * 2,
                "flops": 4 * visible * case["heads"] * d}
    # one read of the logits; a difference, an exponential and two sums per logit
    return {"bytes": case["rows"] * (case["vocab"] * _BYTES[case["dtype"]] + 16), "flops": 4 * case["rows"] * case["vocab"]}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _quantise(x):
    """[.., D] -> (e4m3 [.., D], exponent bytes [..]): a power-of-two scale for
    each vector, the least that brings its largest magnitude to 448 or below."""
    x = x.float()
    mantissa, exponent = torch.frexp(x.abs().amax(-1))
    e = exponent - 9 + (mantissa > _E4M3_MAX / 512).to(exponent.dtype)
    e = torch.where(mantissa == 0, torch.zeros_like(e), e.clamp(min=-126))
    scaled = x * torch.exp2(-e.float())[..., None]
    return scaled.to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _dequantise(q, exponents):
    return q.float() * torch.exp2(exponents.float() - 127.0)[..., None]


def _make_pages(case, gen, lengths, filled):
    """A pool of pages handed out in shuffled order, and the block table."""
    dev, page = "cuda", case["page"]
    need = [max(1, -(-n // page)) for n in lengths]
    spare = 3
    order = list(range(sum(need) + spare))
    random.Random(sum(need)).shuffle(order)
    table = torch.zeros((len(lengths), max(need)), dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    shape = (len(order), case["kv_heads"], page, case["head_dim"])
    pages, scales = [], []
    for _ in range(2):
        if filled:
            x = torch.randn(shape, generator=gen, device=dev, dtype=_DTYPES[case["dtype"]])
            if case["stored"] == "e4m3":
                q, s = _quantise(x)
                pages.append(q)
                scales.append(s)
            else:
                pages.append(x)
        elif case["stored"] == "e4m3":
            pages.append(torch.zeros(shape, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn))
            scales.append(torch.full(shape[:3], 127, dtype=torch.uint8, device=dev))
        else:
            pages.append(torch.zeros(shape, dtype=_DTYPES[case["dtype"]], device=dev))
    out = dict(key_pages=pages[0], value_pages=pages[1], table=table.to(dev),
               key_scales=scales[0] if scales else None, value_scales=scales[1] if scales else None)
    if own:
        from oslo_amd import PagedKV
        out["cache"] = PagedKV(out["key_pages"], out["value_pages"], out["table"], out["key_scales"],
                               out["value_scales"])
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"
    state = dict(case=case)
    if case["op"] == "packed":
        lengths = _lengths(case)
        tokens, d, dt = sum(lengths), case["head_dim"], _DTYPES[case["dtype"]]
        state["lengths"] = lengths
        state["scale"] = 1.0 / math.sqrt(d)
        state["q"] = torch.randn((tokens, case["heads"], d), generator=gen, device=dev, dtype=dt)
        state["k"] = torch.randn((tokens, case["kv_heads"], d), generator=gen, device=dev, dtype=dt)
        state["v"] = torch.randn((tokens, case["kv_heads"], d), generator=gen, device=dev, dtype=dt)
        if case["grad"]:
            state["grad"] = torch.randn((tokens, case["heads"], d), generator=gen, device=dev, dtype=dt)
            for name in "qkv":
                state[name].requires_grad_(True)
        if own:
            from oslo_amd import PackedSequences
            state["packed"] = PackedSequences(lengths, dev)
    elif case["op"] == "cache":
        lengths = _lengths(case)
        state.update(_make_pages(case, gen, lengths, filled=False))
        if case["step"]:  # every sequence's newest token
            seqs, positions = list(range(len(lengths))), [n - 1 for n in lengths]
        else:
            seqs = [i for i, n in enumerate(lengths) for _ in range(n)]
            positions = [p for n in lengths for p in range(n)]
        state["seqs"] = torch.tensor(seqs, dtype=torch.int32, device=dev)
        state["positions"] = torch.tensor(positions, dtype=torch.int32, device=dev)
        shape = (len(seqs), case["kv_heads"], case["head_dim"])
        state["k"] = torch.randn(shape, generator=gen, device=dev, dtype=_DTYPES[case["dtype"]])
        state["v"] = torch.randn(shape, generator=gen, device=dev, dtype=_DTYPES[case["dtype"]])
    elif case["op"] == "decode":
        lengths = _lengths(case)
        state.update(_make_pages(case, gen, lengths, filled=True))
        state["host_lengths"] = lengths
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=dev)
        state["scale"] = 1.0 / math.sqrt(case["head_dim"])
        state["q"] = torch.randn((len(lengths), case["heads"], case["head_dim"]), generator=gen, device=dev,
                                 dtype=_DTYPES[case["dtype"]])
    else:
        rows, vocab = case["rows"], case["vocab"]
        logits = torch.randn((rows, vocab), generator=gen, device=dev) * 2.0
        # a few dozen candidates stand out, as a language model's do
        some = min(vocab, 32)
        at = torch.randint(0, vocab, (rows, some), generator=gen, device=dev)
        logits.scatter_add_(1, at, 9.0 * torch.rand((rows, some), generator=gen, device=dev))
        if case["banned"]:
            at = torch.randint(0, vocab, (rows, case["banned"]), generator=gen, device=dev)
            logits.scatter_(1, at, float("-inf"))
        state["logits"] = logits.to(_DTYPES[case["dtype"]])
        state["u"] = torch.rand((rows,), generator=gen, device=dev)
        settings = dict(temperature=case["temperature"], top_k=case["top_k"], top_p=case["top_p"], min_p=case["min_p"])
        if case["per_row"]:
            r = torch.rand((4, rows), generator=gen, device=dev)
            settings["temperature"] = (case["temperature"] * (0.5 + r[0])).float()
            settings["top_k"] = torch.where(r[1] < 0.5, torch.full_like(r[1], float(case["top_k"])),
                                            1.0 + torch.floor(r[1] * min(vocab, 200))).to(torch.int32)
            settings["top_p"] = torch.where(r[2] < 0.3, torch.ones_like(r[2]), case["top_p"] * r[2])
            settings["min_p"] = torch.where(r[3] < 0.5, torch.zeros_like(r[3]), case["min_p"] * r[3])
        state["settings"] = settings
    return state


# ---------------------------------------------------------------------------
# the operators in elementary operations
# ---------------------------------------------------------------------------

def _plain_packed(state):
    case = state["case"]
    heads, groups, window = case["heads"], case["heads"] // case["kv_heads"], case["window"]
    q, k, v = state["q"].detach(), state["k"].detach(), state["v"].detach()
    out = torch.empty_like(q)
    grads = [torch.empty_like(t) for t in (q, k, v)] if case["grad"] else []
    start = 0
    for n in state["lengths"]:
        rows = slice(start, start + n)
        start += n
        qs = q[rows].float().transpose(0, 1).contiguous()
        ks = k[rows].float().transpose(0, 1).repeat_interleave(groups, 0).contiguous()
        vs = v[rows].float().transpose(0, 1).repeat_interleave(groups, 0).contiguous()
        at = torch.arange(n, device=q.device)
        hidden = at[None, :] > at[:, None]
        if window:
            hidden = hidden | (at[None, :] <= at[:, None] - window)
        s = torch.matmul(qs, ks.transpose(1, 2).contiguous()) * state["scale"]
        s.masked_fill_(hidden, float("-inf"))
        p = torch.exp(s - s.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        o = torch.matmul(p, vs)
        out[rows] = o.transpose(0, 1).to(out.dtype)
        if case["grad"]:
            g = state["grad"][rows].float().transpose(0, 1).contiguous()
            dv = torch.matmul(p.transpose(1, 2).contiguous(), g)
            dp = torch.matmul(g, vs.transpose(1, 2).contiguous())
            ds = p * (dp - (g * o).sum(-1, keepdim=True)) * state["scale"]
            dq = torch.matmul(ds, ks)
            dk = torch.matmul(ds.transpose(1, 2).contiguous(), qs)
            dk = dk.view(heads // groups, groups, n, -1).sum(1)
            dv = dv.view(heads // groups, groups, n, -1).sum(1)
            for grad, value in zip(grads, (dq, dk, dv)):
                grad[rows] = value.transpose(0, 1).to(grad.dtype)
    return [out] + grads


def _plain_cache(state):
    case, page = state["case"], state["case"]["page"]
    positions = state["positions"].long()
    ids = state["table"][state["seqs"].long(), positions // page].long()
    slots = positions % page
    if case["stored"] != "e4m3":
        state["key_pages"][ids, :, slots] = state["k"]
        state["value_pages"][ids, :, slots] = state["v"]
        return [state["key_pages"], state["value_pages"]]
    out = []
    for name, x in (("key", state["k"]), ("value", state["v"])):
        q, exponents = _quantise(x)
        pages, scales = state[name + "_pages"].view(torch.uint8), state[name + "_scales"]
        pages[ids, :, slots] = q.view(torch.uint8)
        scales[ids, :, slots] = exponents
        back = _dequantise(pages[ids, :, slots].view(torch.float8_e4m3fn), scales[ids, :, slots])
        out.append(back.to(x.dtype))
    return out


def _plain_decode(state):
    case, page = state["case"], state["case"]["page"]
    groups = case["heads"] // case["kv_heads"]
    out = torch.empty_like(state["q"])
    for i, n in enumerate(state["host_lengths"]):
        first = max(0, n - case["window"]) if case["window"] else 0
        ids = state["table"][i, first // page:-(-n // page)].long()
        skip = first - first // page * page
        kv = []
        for name in ("key", "value"):
            x = state[name + "_pages"]
            x = x.view(torch.uint8)[ids].view(x.dtype) if case["stored"] == "e4m3" else x[ids]
            x = _dequantise(x, state[name + "_scales"][ids]) if case["stored"] == "e4m3" else x.float()
            kv.append(x.transpose(0, 1).reshape(case["kv_heads"], -1, case["head_dim"])[:, skip:skip + n - first])
        q = state["q"][i].float().view(case["kv_heads"], groups, -1)
        s = torch.matmul(q, kv[0].transpose(1, 2).contiguous()) * state["scale"]
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.matmul(p / p.sum(-1, keepdim=True), kv[1].contiguous())
        out[i] = o.reshape(case["heads"], -1).to(out.dtype)
    return [out]


def _column(value, like):
    """A setting as a column of 64-bit numbers, one per row."""
    if isinstance(value, torch.Tensor):
        return value.double()[:, None]
    return torch.full((like.shape[0], 1), float(value), dtype=torch.float64, device=like.device)


def _plain_sample(state):
    # (in 64 bits: tokens next to a border of the filters or of the draw have to come out right)
    s, logits = state["settings"], state["logits"]
    vocab = logits.shape[1]
    x = logits.double() / _column(s["temperature"], logits)
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    mass = torch.exp(x - x[:, :1])
    rank = torch.arange(vocab, device=x.device)[None, :]
    top_k = _column(s["top_k"], logits)
    mass = mass * ((rank < top_k) | (top_k <= 0))
    top_p = _column(s["top_p"], logits)
    run = torch.cumsum(mass, 1)
    keep = (run - mass < top_p * run[:, -1:]) | (top_p >= 1)
    keep = keep & (mass >= _column(s["min_p"], logits))
    mass = torch.zeros_like(mass).scatter_(1, order, mass * keep)
    run = torch.cumsum(mass, 1)
    token = (run <= state["u"].double()[:, None] * run[:, -1:]).sum(1, keepdim=True)
    logprob = torch.log(mass.gather(1, token) / run[:, -1:])
    return [token[:, 0], logprob[:, 0].float()]


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"packed": _plain_packed, "cache": _plain_cache, "decode": _plain_decode,
                "sample": _plain_sample}[op](state)
    import oslo_amd
    if op == "packed":
        window = state["case"]["window"] or None
        out = oslo_amd.FusedPackedAttention.apply(state["q"], state["k"], state["v"], state["packed"], state["scale"],
                                                  window)
        if not state["case"]["grad"]:
            return [out]
        return [out.detach()] + list(torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["grad"]))
    if op == "cache":
        cache = state["cache"]
        oslo_amd.FusedPagedKV.write(cache, state["k"], state["v"], state["seqs"], state["positions"])
        if state["case"]["stored"] != "e4m3":
            return [cache.key_pages, cache.value_pages]
        return list(oslo_amd.FusedPagedKV.read(cache, state["seqs"], state["positions"], state["k"].dtype))
    if op == "decode":
        return [oslo_amd.FusedPagedDecodeAttention.apply(state["q"], state["cache"], state["lengths"], state["scale"],
                                                         state["case"]["window"] or None)]
    return list(oslo_amd.FusedSampling.apply(state["logits"], state["u"], **state["settings"]))


# ---------------------------------------------------------------------------
# the results in 64 bits
# ---------------------------------------------------------------------------

def _exact_attention(q, k, v, scale, first, last, grad=None):
    """One head: rows of q [n, D] against the keys first[i] .. last[i] of k, v
    [m, D]; with grad [n, D] also the three gradients. All 64-bit."""
    at = torch.arange(k.shape[0], device=k.device)
    seen = (at[None, :] >= first[:, None]) & (at[None, :] <= last[:, None])
    s = (q @ k.t()) * scale
    p = torch.softmax(s.masked_fill(~seen, -math.inf), dim=1)
    o = p @ v
    if grad is None:
        return o, None, None, None
    dp = grad @ v.t()
    ds = scale * p * (dp - (dp * p).sum(1, keepdim=True))
    return o, ds @ k, ds.t() @ q, p.t() @ grad


def _exact_packed(case, state):
    groups = case["heads"] // case["kv_heads"]
    q, k, v = (state[name].detach() for name in "qkv")
    outs = [torch.zeros(q.shape, dtype=torch.float64, device=q.device)]
    if case["grad"]:
        outs += [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (q, k, v)]
    start = 0
    for n in state["lengths"]:
        rows = slice(start, start + n)
        start += n
        last = torch.arange(n, device=q.device)
        first = last - case["window"] + 1 if case["window"] else torch.zeros_like(last)
        for h in range(case["heads"]):
            kv = h // groups
            g = state["grad"][rows, h].double() if case["grad"] else None
            o, dq, dk, dv = _exact_attention(q[rows, h].double(), k[rows, kv].double(), v[rows, kv].double(),
                                             state["scale"], first, last, g)
            outs[0][rows, h] = o
            if case["grad"]:
                outs[1][rows, h] = dq
                outs[2][rows, kv] += dk
                outs[3][rows, kv] += dv
    return outs


def _exact_cache(case, state):
    outs = []
    for name, x in (("key", state["k"]), ("value", state["v"])):
        if case["stored"] != "e4m3":
            pages = state[name + "_pages"].double()
            for t, (s, p) in enumerate(zip(state["seqs"].tolist(), state["positions"].tolist())):
                pages[int(state["table"][s, p // case["page"]]), :, p % case["page"]] = x[t].double()
            outs.append(pages)
            continue
        x = x.double().cpu().numpy()
        # the least e with amax <= 448 * 2^e, then the nearest multiple of the step at each value's size (ties to even)
        amax = np.abs(x).max(-1, keepdims=True)
        e = np.ceil(np.log2(np.where(amax > 0, amax, _E4M3_MAX) / _E4M3_MAX))
        e = np.where(amax > _E4M3_MAX * 2.0 ** e, e + 1, np.where(amax <= _E4M3_MAX * 2.0 ** (e - 1), e - 1, e))
        y = x / 2.0 ** e
        step = 2.0 ** (np.clip(np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -20))), -6, 8) - 3)
        outs.append(torch.from_numpy(np.rint(y / step) * step * 2.0 ** e))
    return outs


def _exact_decode(case, state):
    groups, page = case["heads"] // case["kv_heads"], case["page"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    for i, n in enumerate(state["host_lengths"]):
        at = torch.arange(max(0, n - case["window"]) if case["window"] else 0, n, device="cuda")
        ids, slots = state["table"][i].long()[at // page], at % page
        kv = []
        for name in ("key", "value"):
            x = state[name + "_pages"]
            x = (x.view(torch.uint8)[ids, :, slots].view(x.dtype) if case["stored"] == "e4m3" else x[ids, :, slots])
            x = x.double() if case["stored"] != "e4m3" else x.float().double()
            if case["stored"] == "e4m3":
                x = x * 2.0 ** (state[name + "_scales"][ids, :, slots].double() - 127.0)[..., None]
            kv.append(x)
        for h in range(case["kv_heads"]):
            rows = slice(h * groups, (h + 1) * groups)
            w = torch.softmax(state["q"][i, rows].double() @ kv[0][:, h].t() * state["scale"], dim=1)
            out[i, rows] = w @ kv[1][:, h]
    return [out]


def _exact_sample(case, state):
    logits, u = state["logits"].double().cpu().numpy(), state["u"].double().cpu().numpy()
    rows, vocab = logits.shape
    settings = {}
    for name, value in state["settings"].items():
        settings[name] = value.double().cpu().numpy() if isinstance(value, torch.Tensor) else np.full(rows, float(value))
    tokens, logprobs = np.zeros(rows, dtype=np.int64), np.zeros(rows)
    for i in range(rows):
        x = logits[i] / settings["temperature"][i]
        w = np.exp(x - x.max())
        kept = np.flatnonzero(w > 0)
        kept = kept[np.argsort(-x[kept], kind="stable")]
        k = int(settings["top_k"][i])
        if k > 0:
            kept = kept[:k]
        p = settings["top_p"][i]
        if p < 1:
            run = np.cumsum(w[kept].astype(np.longdouble))
            kept = kept[:max(1, int(np.searchsorted(run, np.longdouble(p) * run[-1], side="left")) + 1)]
        kept = np.sort(kept[w[kept] >= settings["min_p"][i]])
        run = np.cumsum(w[kept].astype(np.longdouble))
        j = int(np.searchsorted(run, np.longdouble(u[i]) * run[-1], side="right"))
        tokens[i] = kept[j]
        logprobs[i] = float(np.log(w[kept[j]] / run[-1]))
    return [torch.from_numpy(tokens), torch.from_numpy(logprobs)]


def exact(case, seed):
    state = prepare(case, seed)
    return {"packed": _exact_packed, "cache": _exact_cache, "decode": _exact_decode,
            "sample": _exact_sample}[case["op"]](case, state)
