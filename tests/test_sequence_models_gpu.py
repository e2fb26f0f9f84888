"""The models over sequences of different lengths: a packed training forward and
backward, and generation from a list of prompts (packed prompts, the paged cache
in 16 and 8 bits, the paged decoding steps, sampling), against the unfused model
in 64 bits run on one sequence at a time.

Tolerances of the model runs: a packed (or paged) run rounds to 16 bits at the
places where the fused model rounds when it takes one sequence at a time, so the
norms of the two runs' errors estimate the same sum of variances, over
thousands of values; one may exceed the other by half at most (``ALIKE``)."""

import pytest
import torch

from oslo_amd import (FusedPagedKV, FusedSampling, GPT2Config, GPT2LMHeadModel, GPTJConfig, GPTJForCausalLM,
                      GPTNeoConfig, GPTNeoForCausalLM, PackedSequences, PagedState)
from oslo_amd.generation_utils import PagedDecoder
from oslo_amd.sequences import PagedLayer

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
VOCAB, POSITIONS = 331, 320
FAMILIES = ["gpt2", "gptj", "gpt_neo"]
ALIKE = 1.5
LENGTHS = [37, 1, 200, 128, 64]


def make(family, layers=2, dtype=torch.float16, seed=0):
    """(fused model of ``dtype`` on the device, the unfused one in 64 bits on the host)."""
    torch.manual_seed(seed)
    if family == "gpt2":
        cls, cfg = GPT2LMHeadModel, GPT2Config(vocab_size=VOCAB, n_positions=POSITIONS, n_embd=128, n_layer=layers,
                                               n_head=2, resid_pdrop=0.0, embd_pdrop=0.0, attn_pdrop=0.0)
    elif family == "gptj":
        cls, cfg = GPTJForCausalLM, GPTJConfig(vocab_size=VOCAB, n_positions=POSITIONS, n_embd=256, n_layer=layers,
                                               n_head=2, rotary_dim=32)
    else:
        cls, cfg = GPTNeoForCausalLM, GPTNeoConfig(vocab_size=VOCAB, max_position_embeddings=POSITIONS, hidden_size=128,
                                                   num_layers=layers, num_heads=2, window_size=24,
                                                   attention_layers=["local", "global"][:layers])
    model = cls(cfg).eval()
    with torch.no_grad():
        for p in model.parameters():
            if p.dim() > 1:
                p.mul_(4.0)  # attention that is far from uniform, logits far from equal
            p.copy_(p.to(dtype))
    plain = cls(cfg).eval()
    plain.load_state_dict(model.state_dict())
    return model.to(dtype).to(DEV).fuse(), plain.double()


def tokens(n, seed):
    return torch.randint(0, VOCAB, (n,), generator=torch.Generator().manual_seed(seed))


def norm_error(got, want):
    return float((got.detach().double().cpu() - want).norm() / want.norm())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("family", FAMILIES)
def test_packed_forward_and_gradients(family, dtype):
    model, plain = make(family, dtype=dtype)
    lengths, extra = [37, 1, 200, 0, 128, 64], 5
    packed = PackedSequences(lengths, DEV)
    ids = tokens(packed.total + extra, 1)
    pieces = [p for p in ids[:packed.total].split(lengths) if len(p)]
    count = sum(len(p) - 1 for p in pieces)

    def summed(m, run):
        """Loss over one sequence at a time; gradients are left in the parameters."""
        loss = 0.0
        for p in pieces:
            logits = run(m, p)
            if len(p) > 1:
                part = torch.nn.functional.cross_entropy(
                    logits[:-1].to(torch.float64 if m is plain else torch.float32), p[1:].to(logits.device),
                    reduction="sum") / count
                part.backward()
                loss += float(part.detach())
        return loss

    want_loss = summed(plain, lambda m, p: m(p[None])["logits"][0])
    want = torch.cat([p.grad.flatten() for p in plain.parameters() if p.grad is not None])
    names = [n for n, p in plain.named_parameters() if p.grad is not None]
    params = dict(model.named_parameters())

    single_loss = summed(model, lambda m, p: m(p[None].to(DEV))["logits"][0])
    single = torch.cat([params[n].grad.flatten() for n in names])
    model.zero_grad()
    out = model(ids[None].to(DEV), labels=ids[None].to(DEV), packed=packed)
    out["loss"].backward()
    got = torch.cat([params[n].grad.flatten() for n in names])

    with torch.no_grad():
        logits = torch.cat([plain(p[None])["logits"][0] for p in pieces])
        alone = torch.cat([model(p[None].to(DEV))["logits"][0] for p in pieces])
    assert out["logits"].shape == (1, packed.total + extra, VOCAB) and out["logits"].isfinite().all()
    assert norm_error(out["logits"][0, :packed.total], logits) <= ALIKE * norm_error(alone, logits)
    # (the loss is a mean over some 400 tokens of logits that are off by the norms above)
    assert abs(float(out["loss"].detach()) - want_loss) <= norm_error(alone, logits) * float(logits.abs().max())
    assert abs(single_loss - want_loss) <= norm_error(alone, logits) * float(logits.abs().max())
    assert got.isfinite().all()
    assert norm_error(got, want) <= ALIKE * norm_error(single, want)


def test_packed_row_gives_each_sequence_the_same_bits_wherever_it_lies():
    """No sequence sees another: other neighbours, the same result (the products take the same row count)."""
    model, _ = make("gpt2")
    a, b, c = tokens(100, 1), tokens(77, 2), tokens(77, 3)
    with torch.no_grad():
        one = model(torch.cat([a, b])[None].to(DEV), packed=PackedSequences([100, 77], DEV))["logits"][0]
        two = model(torch.cat([a, c])[None].to(DEV), packed=PackedSequences([100, 77], DEV))["logits"][0]
    assert torch.equal(one[:100], two[:100]) and not torch.equal(one[100:], two[100:])


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
@pytest.mark.parametrize("family", FAMILIES)
def test_prompts_and_steps_over_the_paged_cache(family, graph):
    """Logits behind the prompts and behind each of the steps, one sequence being full before the others."""
    model, plain = make(family)
    prompts = [tokens(n, 10 + i) for i, n in enumerate(LENGTHS)]
    capacity, steps = 204, 9
    feed = torch.stack([tokens(steps, 30 + i) for i in range(len(LENGTHS))])
    got, alone, want = [], [], []
    with torch.no_grad():
        decoder = PagedDecoder(model, [p.to(DEV) for p in prompts], capacity, graph, False)
        rows = [decoder.prompt().clone()]
        for step in range(steps):
            rows.append(decoder.step(feed[:, step].to(DEV)).clone())
        for i, p in enumerate(prompts):
            new = min(steps, capacity - len(p))
            whole = torch.cat([p, feed[i, :new]])[None]
            want.append(plain(whole)["logits"][0, len(p) - 1:])
            alone.append(model(whole.to(DEV))["logits"][0, len(p) - 1:])
            got.append(torch.stack([r[i] for r in rows[:new + 1]]))
    assert all(r.isfinite().all() for r in rows)
    want, alone, got = torch.cat(want), torch.cat(alone), torch.cat(got)
    assert norm_error(got, want) <= ALIKE * norm_error(alone, want)
    assert decoder.state.lengths.tolist() == [min(n + steps, capacity - 1) for n in LENGTHS]


class PlainLayer(PagedLayer):
    """The cache is written and read back by the kernels, the attention is spelled out in 64 bits."""

    def attend(self, query, key, value, scale, window=None):
        state = self.state
        FusedPagedKV.write(self.cache, key, value, state.rows, state.lengths)
        out = torch.empty_like(query)
        for i, n in enumerate(state.visible.tolist()):
            at = torch.arange(0 if window is None else max(0, n - window), n, dtype=torch.int32, device=query.device)
            k, v = FusedPagedKV.read(self.cache, torch.full_like(at, i), at, query.dtype)
            w = torch.softmax((query[i].double().unsqueeze(0) * k.double()).sum(-1) * scale, dim=0)
            out[i] = (w.unsqueeze(-1) * v.double()).sum(0).to(query.dtype)
        return out


@pytest.mark.parametrize("family", FAMILIES)
def test_steps_over_an_8_bit_cache(family):
    """One layer, so that both runs put the same numbers into their caches: the logits differ by the rounding of
    an attention output (half a step of fp16 each) passed through the rest of the layer, as those of the fused
    model differ from the 64-bit model's, where there are more roundings."""
    model, plain = make(family, layers=1)
    prompts = [tokens(n, 10 + i).to(DEV) for i, n in enumerate(LENGTHS)]
    with torch.no_grad():
        whole = prompts[2][None]
        one_run = norm_error(model(whole)["logits"][0], plain(whole.cpu())["logits"][0])
        runs = []
        for layer in (PagedLayer, PlainLayer):
            decoder = PagedDecoder(model, prompts, 256, False, True)
            state, rows = decoder.state, [decoder.prompt().clone()]
            assert all(c.quantized for c in state.caches)
            for step in range(4):
                state.begin_step()
                feed = torch.stack([tokens(4, 30 + i)[step] for i in range(len(LENGTHS))]).to(DEV)[None]
                rows.append(model(feed, past_key_values=[layer(state, c) for c in state.caches])["logits"][0].clone())
                state.end_step()
            runs.append(torch.stack(rows))
    assert torch.equal(runs[0][0], runs[1][0])
    assert norm_error(runs[0][1:], runs[1][1:].double().cpu()) <= ALIKE * 2 ** 0.5 * one_run


@pytest.mark.parametrize("quantized", [False, True], ids=["16bit", "8bit"])
@pytest.mark.parametrize("family", FAMILIES)
def test_generate_from_a_list_of_prompts(family, quantized):
    model, _ = make(family)
    prompts = [tokens(n, 50 + i).to(DEV) for i, n in enumerate([5, 40, 1, 129])]
    kw = dict(max_length=140, quantized_cache=quantized)
    greedy = model.generate(prompts, **kw)
    with torch.no_grad():  # the same by hand
        decoder = PagedDecoder(model, prompts, 140, False, quantized)
        picked = [decoder.prompt().argmax(-1)]
        for _ in range(138):
            picked.append(decoder.step(picked[-1]).argmax(-1))
    picked = torch.stack(picked, 1)
    for i, (p, row) in enumerate(zip(prompts, greedy)):
        assert row.shape == (140,) and row.dtype == p.dtype and torch.equal(row[:len(p)], p)
        assert torch.equal(row[len(p):], picked[i, :140 - len(p)])
    for a, b in zip(greedy, model.generate(prompts, graph=True, **kw)):
        assert torch.equal(a, b)
    for a, b in zip(greedy, model.generate(prompts, do_sample=True, top_k=1, **kw)):
        assert torch.equal(a, b)
    # an end: the same tokens, cut behind it
    eos = int(greedy[1][60])
    for row, p, cut in zip(greedy, prompts, model.generate(prompts, eos_token_id=eos, **kw)):
        ends = (row[len(p):] == eos).nonzero()
        n = len(p) + int(ends[0]) + 1 if len(ends) else 140
        assert torch.equal(cut, row[:n])
    for p, row in zip(prompts, model.generate(prompts, eos_token_id=eos, min_length=100, **kw)):
        assert len(row) >= 100 and eos not in row[len(p):99].tolist()
    # draws: by the generator alone, eager and captured
    draws = [model.generate(prompts, do_sample=True, temperature=1.3, top_p=0.9, graph=graph,
                            generator=torch.Generator(DEV).manual_seed(seed), **kw)
             for graph, seed in ((False, 1), (True, 1), (False, 2))]
    assert all(torch.equal(a, b) for a, b in zip(draws[0], draws[1]))
    assert not all(torch.equal(a, b) for a, b in zip(draws[0], draws[2]))


def test_generate_draws_from_equal_prompts():
    model, _ = make("gpt2")
    ids = torch.stack([tokens(9, i) for i in range(3)]).to(DEV)
    greedy = model.generate(ids, max_length=30)
    assert torch.equal(model.generate(ids, max_length=30, do_sample=True, top_k=1), greedy)
    assert torch.equal(model.generate(ids, max_length=30, do_sample=True, temperature=0.0), greedy)
    kw = dict(max_length=30, do_sample=True, top_p=0.8, temperature=1.2, no_repeat_ngram_size=2)
    drawn = [model.generate(ids, generator=torch.Generator(DEV).manual_seed(3), graph=graph, **kw)
             for graph in (False, False, True)]
    assert torch.equal(drawn[0], drawn[1]) and drawn[2].shape == (3, 30)
    for row in drawn[0].tolist():
        pairs = list(zip(row[8:], row[9:]))
        assert len(set(pairs)) == len(pairs)
    u = torch.rand(3, generator=torch.Generator(DEV).manual_seed(3), device=DEV)
    with torch.no_grad():
        logits = model(ids)["logits"][:, -1].float()
    first = FusedSampling.apply(logits, u, temperature=1.2, top_p=0.8)[0]
    kw.pop("no_repeat_ngram_size")
    again = model.generate(ids, generator=torch.Generator(DEV).manual_seed(3), **kw)
    assert torch.equal(again[:, 9], first)


def test_a_captured_packed_training_step():
    """Forward and backward of a packed row captured into a graph and replayed between eager work."""
    model, _ = make("gptj")
    model.train()
    packed = PackedSequences([70, 130, 3], DEV)
    ids = tokens(packed.total, 1)[None].to(DEV)
    params = [p for p in model.parameters() if p.requires_grad]

    def step():
        for p in params:
            p.grad = None
        loss = model(ids, labels=ids, packed=packed)["loss"]
        loss.backward()
        return loss.detach()

    def eager(row):
        ids.copy_(row)
        loss = step()
        return loss.clone(), [p.grad.clone() for p in params if p.grad is not None]

    rows = [tokens(packed.total, seed)[None].to(DEV) for seed in (1, 2, 3)]
    wants = [eager(r) for r in rows]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    for p in params:
        p.grad = None
    with torch.cuda.graph(graph):
        loss = step()
    grads = [p.grad for p in params if p.grad is not None]
    for row, (want_loss, want) in zip(rows, wants):
        ids.copy_(row)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.allclose(loss, want_loss, rtol=2.0 ** -10, atol=0.0)
        for g, w in zip(grads, want):
            # (torch's embedding gradients add in any order)
            assert float((g.float() - w.float()).norm()) <= 2.0 ** -8 * float(w.float().norm()) + 1e-6


def test_devices_of_a_state_and_a_model_must_agree():
    model, _ = make("gpt2", layers=1)
    state = PagedState([0, 0], 8, 1, 2, 64, torch.bfloat16, DEV)
    with pytest.raises(RuntimeError, match="cache"), torch.no_grad():
        model(torch.zeros((1, 2), dtype=torch.long, device=DEV), past_key_values=state.begin_step())


@pytest.mark.parametrize("family", FAMILIES)
def test_a_prompt_that_fills_the_cache_is_followed_by_steps(family):
    """The model's last position, and the cache's: the next tokens overwrite it, as they do once a sequence has grown
    to be full."""
    model, _ = make(family)
    prompts = [tokens(n, 70 + i).to(DEV) for i, n in enumerate([POSITIONS, 5])]
    feed = torch.stack([tokens(3, 80 + i) for i in range(2)]).to(DEV)
    rows = []
    with torch.no_grad():
        for first in (POSITIONS, POSITIONS - 1):  # (the position the first step writes, either way)
            state = PagedState([first, 5], POSITIONS, len(model.transformer.h), 2, 128 if family == "gptj" else 64,
                               torch.float16, DEV)
            packed = PackedSequences([len(p) for p in prompts], DEV)
            model.transformer(torch.cat(prompts)[None], None, state.prompt_layers(packed))
            rows.append([])
            for step in range(3):
                logits = model(feed[None, :, step], past_key_values=state.begin_step())["logits"][0]
                state.end_step()
                rows[-1].append(logits.clone())
        assert state.lengths.tolist() == [POSITIONS - 1, 8]
    for a, b in zip(*rows):
        assert a.isfinite().all() and torch.equal(a, b)


def forget_rotary_tables():
    """Other lengths are asked for until the last tables have gone, and memory of their size is written over."""
    from oslo_amd.modeling_gptj import rotary_tables
    for n in range(700, 720):
        rotary_tables(32, n, torch.device(DEV))
    return [torch.full((n, 16), float("nan"), device=DEV) for n in range(8, 400, 8) for _ in range(4)]


def test_captured_graphs_keep_their_rotary_tables():
    """A captured decoding step over paged and static caches and a captured forward, replayed after the tables of many
    other lengths have been made."""
    model, _ = make("gptj")
    ids = tokens(60, 5)[None].to(DEV)
    with torch.no_grad():
        state = PagedState([9, 30], 40, len(model.transformer.h), 2, 128, torch.float16, DEV)
        packed = PackedSequences([9, 30], DEV)
        feed = torch.stack([tokens(2, i) for i in (1, 2)]).to(DEV)
        forget_rotary_tables()

        def step():
            return model(feed[:1], past_key_values=state.begin_step())["logits"]

        def row():
            return model(ids[:, :39], packed=packed)["logits"]

        def dense():
            return model(ids[:, :45])["logits"]
        model.transformer(ids[:, :39], None, state.prompt_layers(packed))
        for run in (step, row, dense):
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                run()
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = run()
            junk = forget_rotary_tables()
            for _ in range(3):
                want = run().clone()
                forget_rotary_tables()
                graph.replay()
                torch.cuda.synchronize()
                assert want.isfinite().all() and torch.equal(out, want)
            del junk
        # a graph that generate() keeps
        first = model.generate(ids[:, :20], max_length=50, static_cache=True, graph=True)
        junk = forget_rotary_tables()
        assert torch.equal(model.generate(ids[:, :20], max_length=50, static_cache=True, graph=True), first)
        del junk


def test_rotary_tables_made_inside_a_capture_are_not_handed_on():
    """Without a warm-up the tables are filled by the replays alone."""
    from oslo_amd.modeling_gptj import rotary_tables
    device = torch.device(DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made = rotary_tables(32, 333, device)
    other = rotary_tables(32, 333, device)
    want = torch.sin(torch.arange(333.0)[:, None] / 10000 ** (torch.arange(0, 32, 2.0) / 32))
    assert (other[0].cpu() - want).abs().max() < 1e-4
    for _ in range(3):
        made[0].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(made[0], other[0]) and torch.equal(made[1], other[1])


@pytest.mark.parametrize("family", FAMILIES)
def test_a_capture_is_the_first_to_use_packed_sequences(family):
    """Made before the capture, but used by nobody: positions, owners and last tokens of prompts that go into the cache."""
    model, _ = make(family)
    lengths = [37, 1, 60]
    ids = tokens(sum(lengths), 3)[None].to(DEV)

    def prompts(packed, state):
        h = model.transformer(ids, None, state.prompt_layers(packed))[0][0]
        return model.lm_head(h.index_select(0, packed.last_tokens()))

    def fresh():
        return (PackedSequences(lengths, DEV), PagedState(lengths, 64, len(model.transformer.h), 2,
                                                          128 if family == "gptj" else 64, torch.float16, DEV))
    with torch.no_grad():
        packed, state = fresh()
        want = prompts(packed, state)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            prompts(*fresh())
        torch.cuda.current_stream().wait_stream(side)
        other, caches = fresh()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = prompts(other, caches)
        for seed in (3, 4, 5):
            ids.copy_(tokens(sum(lengths), seed)[None])
            graph.replay()
            want = prompts(packed, state)
            torch.cuda.synchronize()
            assert torch.equal(got, want)
            for a, b in zip(state.caches, caches.caches):
                assert torch.equal(a.key_pages, b.key_pages) and torch.equal(a.value_pages, b.value_pages)
