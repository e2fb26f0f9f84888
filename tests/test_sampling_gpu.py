"""Sampling (temperature, top-k, top-p, min-p, the draw) against plain code in
float64. Tokens are whole numbers and have to be the same: the kernel's masses
are whole multiples of 2^(ceil(log2 V) - 62) of the largest, the plain code's
float64 sums are off by less, and no case here puts a border closer than that to
a sum unless the sums are exact in both (equal logits). Log-probabilities are
one fp32 rounding of a value computed in 64 bits: 2^-24 relative, 2^-40 for the
masses' rounding, taken as 1.1 * 2^-24 |x| + 2^-40."""

import itertools

import pytest
import torch

from oslo_amd import FusedSampling
from tests.util import IDS, randn

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def plain(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    rows, vocab = logits.shape
    dev = logits.device

    def column(x):
        x = x.double() if isinstance(x, torch.Tensor) else torch.full((rows,), float(x), dtype=torch.float64, device=dev)
        return x[:, None]
    x = logits.double().nan_to_num(nan=-float("inf"), posinf=float("inf"), neginf=-float("inf"))
    t = column(temperature)
    top = x.amax(1, keepdim=True)
    greedy = ~(t > 0)
    depth = torch.where(x == top, torch.zeros_like(x), (x - top) / torch.where(greedy, torch.ones_like(t), t))
    order = torch.sort(x, dim=1, descending=True, stable=True)[1]
    mass = torch.exp(depth).gather(1, order)
    rank = torch.arange(vocab, device=dev)[None, :]
    k = torch.where(greedy, torch.ones_like(t), column(top_k))
    mass = mass * ((rank < k) | (k <= 0))
    run = torch.cumsum(mass, 1)
    p = torch.where(greedy, torch.ones_like(t), column(top_p))
    keep = (run - mass < p * run[:, -1:]) | (p >= 1)
    keep |= rank == 0
    mass = mass * keep * (mass >= torch.where(greedy, torch.zeros_like(t), column(min_p)))
    mass = torch.zeros_like(mass).scatter_(1, order, mass)
    run = torch.cumsum(mass, 1)
    token = (run <= u.double()[:, None] * run[:, -1:]).sum(1, keepdim=True)
    return token[:, 0], torch.log(mass.gather(1, token) / run[:, -1:])[:, 0]


def check(logits, u, **settings):
    tokens, logprobs = FusedSampling.apply(logits, u, **settings)
    want, want_log = plain(logits, u, **settings)
    assert tokens.dtype == torch.int64 and logprobs.dtype == torch.float32
    wrong = (tokens != want).nonzero()[:, 0].tolist()
    assert not wrong, [(r, tokens[r].item(), want[r].item()) for r in wrong[:5]]
    err = (logprobs.double() - want_log).abs()
    assert (err <= 1.1 * 2.0 ** -24 * want_log.abs() + 2.0 ** -40).all(), err.max()
    return tokens


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=50, temperature=1.3), dict(top_p=0.9),
            dict(top_k=20, top_p=0.5, min_p=0.05, temperature=0.8), dict(min_p=0.1), dict(top_p=0.0), dict(temperature=0.0),
            dict(top_k=10 ** 6, top_p=0.999), dict(top_k=300, min_p=1.0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=IDS.get)
@pytest.mark.parametrize("rows,vocab", [(3, 1), (5, 2), (9, 40), (4, 1000), (2, 8192), (3, 8193), (17, 50257), (2, 70001)])
def test_tokens(rows, vocab, dtype):
    logits = randn((rows, vocab), dtype, seed=vocab, std=2.5).to(DEV)
    u = torch.rand((rows,), generator=torch.Generator().manual_seed(vocab)).to(DEV)
    for settings in SETTINGS:
        check(logits, u, **settings)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=IDS.get)
def test_a_setting_for_every_row(dtype):
    rows, vocab = 64, 5003
    g = torch.Generator().manual_seed(1)
    logits = randn((rows, vocab), dtype, seed=2, std=3.0).to(DEV)
    u, t, p, m = (torch.rand((rows,), generator=g).to(DEV) for _ in range(4))
    k = torch.randint(-3, 200, (rows,), generator=g, dtype=torch.int32).to(DEV)
    t[:5] = 0.0
    check(logits, u, temperature=t * 2, top_k=k, top_p=p * 1.2, min_p=m * 0.2)
    check(logits, u, temperature=0.9, top_k=k, top_p=0.8, min_p=m * 0.2)


def test_equal_logits_go_by_index():
    """Sums of equal masses are exact: u = i / n draws token i, top-k and top-p keep the lowest indices."""
    for vocab in (8, 1024, 50257):
        logits = torch.full((64, vocab), -3.25, device=DEV)
        u = (torch.arange(64, device=DEV) / 64.0)
        tokens = FusedSampling.apply(logits, u)[0]
        assert torch.equal(tokens, torch.floor(u.double() * vocab).long())
        keep = min(vocab, 37)
        tokens = FusedSampling.apply(logits, u, top_k=keep)[0]
        assert torch.equal(tokens, torch.floor(u.double() * keep).long())
        half = -(-vocab // 2)
        tokens = FusedSampling.apply(logits, u, top_p=0.5)[0]
        assert torch.equal(tokens, torch.floor(u.double() * half).long())
    # few distinct values, ties across the cut
    logits = (randn((40, 3001), torch.float32, seed=3).to(DEV) * 2).round()
    u = torch.rand((40,), generator=torch.Generator().manual_seed(9)).to(DEV)
    for k, p in itertools.product((0, 5, 700), (1.0, 0.6)):
        check(logits, u, top_k=k, top_p=p)


def test_infinities_nan_and_rows_of_nothing():
    inf, nan = float("inf"), float("nan")
    logits = torch.tensor([[-inf] * 6, [nan, -inf, nan, -inf, -inf, -inf], [-inf, 2.0, -inf, nan, 2.0, -inf],
                           [1.0, inf, 3.0, inf, -inf, 0.0], [3.0e38, -3.0e38, 0.0, 1.0, 2.0, nan],
                           [nan, 1.0, 1.0, 1.0, 1.0, -inf]], device=DEV)
    u = torch.tensor([0.5, 0.5, 0.75, 0.75, 0.999, 0.3], device=DEV)
    for settings in (dict(), dict(top_k=2), dict(top_p=0.7), dict(min_p=0.5), dict(temperature=0.3), dict(temperature=0.0)):
        tokens, logprobs = FusedSampling.apply(logits, u, **settings)
        assert tokens[:2].tolist() == [-1, -1] and (logprobs[:2] == -inf).all()
        want, want_log = plain(logits[2:], u[2:], **settings)
        assert torch.equal(tokens[2:], want), settings
        assert (logprobs[2:].double() - want_log).abs().max() < 1e-6
    # uniforms at and outside the ends
    logits = torch.zeros((5, 10), device=DEV)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, -1.0, nan], device=DEV)
    assert FusedSampling.apply(logits, u)[0].tolist() == [0, 9, 9, 0, 0]


def test_frequencies_are_the_probabilities():
    logits = torch.tensor([[0.3, -1.0, 2.0, 0.0, 1.5, -4.0, 0.9]], device=DEV)
    n = 20000
    u = (torch.arange(n, device=DEV, dtype=torch.float32) + 0.5) / n
    tokens = FusedSampling.apply(logits.expand(n, 7), u, temperature=0.8)[0]
    p = torch.softmax(logits[0].double() / 0.8, 0)
    assert (torch.bincount(tokens, minlength=7) - n * p).abs().max() <= 1.5


def test_rows_lie_anywhere():
    """Strided rows (the last position of a forward's logits), an odd base address, an odd vocabulary."""
    full = randn((6, 3, 777), torch.bfloat16, seed=11, std=3.0).to(DEV)
    u = torch.rand((6,), generator=torch.Generator().manual_seed(2)).to(DEV)
    view = full[:, -1, :]
    a = FusedSampling.apply(view, u, top_p=0.9)
    b = FusedSampling.apply(view.contiguous(), u, top_p=0.9)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    flat = torch.empty(6 * 777 + 5, dtype=torch.bfloat16, device=DEV)
    for shift in (1, 3, 5):
        odd = flat[shift:shift + 6 * 777].view(6, 777).copy_(view)
        assert torch.equal(FusedSampling.apply(odd, u, top_p=0.9)[0], a[0])
    assert torch.equal(FusedSampling.apply(view.t().contiguous().t(), u, top_p=0.9)[0], a[0])


def test_captured_and_on_another_stream():
    logits = randn((5, 50257), torch.float32, seed=1, std=2.0).to(DEV)
    u = torch.rand((5,), generator=torch.Generator().manual_seed(5)).to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        FusedSampling.apply(logits, u, top_k=40, top_p=0.9)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, logprobs = FusedSampling.apply(logits, u, top_k=40, top_p=0.9)
    for seed in (6, 7, 8):
        u.copy_(torch.rand((5,), generator=torch.Generator().manual_seed(seed)))
        logits.copy_(randn((5, 50257), torch.float32, seed=seed, std=2.0))
        graph.replay()
        torch.cuda.synchronize()
        want = FusedSampling.apply(logits, u, top_k=40, top_p=0.9)
        assert torch.equal(tokens, want[0]) and torch.equal(logprobs, want[1])


def test_refused_calls():
    logits, u = torch.zeros((3, 10), device=DEV), torch.zeros(3, device=DEV)
    for bad in (dict(temperature=-1.0), dict(top_k=-1), dict(top_p=-0.5), dict(min_p=2.0),
                dict(temperature=torch.ones(2, device=DEV)), dict(top_k=torch.ones(3, device=DEV)),
                dict(top_p=torch.ones(3))):
        with pytest.raises(RuntimeError):
            FusedSampling.apply(logits, u, **bad)
    for args in ((logits[0], u), (logits, u[:2]), (logits, u.double()), (logits.long(), u), (logits[:, :0], u)):
        with pytest.raises(RuntimeError):
            FusedSampling.apply(*args)
    assert FusedSampling.apply(logits[:0], u[:0])[0].shape == (0,)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 17, 1000, 5001, 50257])
def test_many_rows_draw_as_few_do(vocab, dtype):
    """Numbers of rows on both sides of the change of block size: the same tokens, the same bits."""
    rows = 260
    g = torch.Generator().manual_seed(vocab)
    logits = (torch.randn((rows, vocab), generator=g) * 3).to(dtype).to(DEV)
    logits[5], logits[6] = 1.0, float("-inf")
    logits[7, vocab // 2:] = float("inf")
    u = torch.rand(rows, generator=g).to(DEV)
    settings = [dict(), dict(top_k=50), dict(top_k=400, top_p=0.9), dict(top_k=3000, top_p=0.95, temperature=0.7),
                dict(top_p=0.92), dict(top_p=0.5, min_p=0.01), dict(min_p=0.1, temperature=1.5), dict(temperature=0.0)]
    for kw in settings:
        many = FusedSampling.apply(logits, u, **kw)
        few = [FusedSampling.apply(logits[i:i + 130], u[i:i + 130], **kw) for i in (0, 130)]
        assert torch.equal(many[0], torch.cat([t for t, _ in few])), kw
        assert torch.equal(many[1], torch.cat([p for _, p in few])), kw


@pytest.mark.parametrize("vocab", [1001, 50257])
def test_logits_as_far_apart_as_the_type_allows(vocab):
    """Differences that overflow 32 bits, in rows that begin anywhere, with and without nothing but -inf beside."""
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn((4, vocab), generator=g)
    logits[0] *= 1.0e38
    logits[0].clamp_(-3.4e38, 3.4e38)
    logits[1, ::7] = -3.4e38
    logits[1, 3] = 3.4e38
    logits[2] = -3.4e38
    logits[2, ::2] = float("-inf")
    logits[3] = float("-inf")
    logits[3, 11:400] = torch.randn(389, generator=g)
    logits, u = logits.to(DEV), torch.rand(4, generator=g).to(DEV)
    for kw in (dict(), dict(top_k=5), dict(top_k=300), dict(top_k=900, top_p=0.7), dict(top_p=0.9), dict(min_p=0.2),
               dict(top_k=50, temperature=1.0e37), dict(top_p=0.5, temperature=1.0e-37)):
        check(logits, u, **kw)


@pytest.mark.parametrize("rows", [4, 260], ids=["few-rows", "many-rows"])
@pytest.mark.parametrize("vocab", [8000, 50257])
def test_top_p_does_not_bring_back_what_top_k_left_out(vocab, rows):
    """More equal logits at top-k's border than the list holds (2048), of which top-p keeps all that top-k
    kept: whole masses of 1, so the plain sums are exact."""
    u = (torch.arange(rows, device=DEV, dtype=torch.float32) + 0.9) / rows
    flat = torch.full((rows, vocab), 0.75, device=DEV)
    some = flat.clone()
    some[:, 5::1000] = 1.5          # a few above the equal ones
    steps = flat.clone()
    steps[:, ::2] = 0.75 - 2.0 ** -20   # two values within a step of the count
    for logits in (flat, some, steps):
        for k in (2049, 3000, 4000):
            for p in (0.5, 0.9999, 0.99999):
                tokens = check(logits, u, top_k=k, top_p=p)
                if logits is flat and p > 0.9:
                    assert torch.equal(tokens, torch.floor(u.double() * k).long())


def test_temperatures_next_to_zero():
    """Positive ones, down to the smallest number there is: the largest logits share the draw (0 takes the first)."""
    logits = torch.tensor([[1.0, 3.0, 2.0, 3.0, -1.0, 3.0], [0.0, -2.0 ** -149, 2.0 ** -149, 0.0, 0.0, 0.0],
                           [-3.0e38, 3.0e38, 3.0e38, 0.0, float("-inf"), float("nan")]], device=DEV)
    for rows in (3, 300):
        x = logits.repeat(rows // 3, 1)
        u = torch.rand((rows,), generator=torch.Generator().manual_seed(3)).to(DEV)
        for t in (5e-324, 1e-310, 1e-306, 7e-306, 1e-300):
            for kw in (dict(), dict(top_k=2), dict(top_p=0.5), dict(min_p=0.5), dict(top_k=4, top_p=0.4, min_p=1.0)):
                tokens = check(x, u, temperature=t, **kw)
                assert tokens[1::3].eq(2).all()
        each = torch.full((rows,), 2.0 ** -149, device=DEV)
        check(x, u, temperature=each, top_p=0.5)
        check(x, u, temperature=2.0 ** -149, top_p=0.5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=IDS.get)
@pytest.mark.parametrize("rows", [3, 257], ids=["few-rows", "many-rows"])
def test_rows_of_as_many_logits_as_are_taken(rows, dtype):
    """500000, and one fewer (rows then begin anywhere). Each mass is off by at most half a unit, 2^-43, so the
    logarithm of their sum by V * 2^-43 / sum; a border of the plain code lies that close to a running sum (some 1e-7
    of the largest mass, where a token's is 1e-3 and more on average) in one draw of ten thousand."""
    for vocab in (500000, 499999):
        g = torch.Generator(DEV).manual_seed(vocab)
        logits = (torch.randn((rows, vocab), generator=g, device=DEV) * 2.5).to(dtype)
        u = torch.rand((rows,), generator=g, device=DEV)
        some = slice(0, 3)
        for kw in (dict(), dict(temperature=0.6, top_k=50), dict(top_k=3000, top_p=0.9), dict(top_p=0.9), dict(min_p=0.01)):
            tokens, logprobs = FusedSampling.apply(logits, u, **kw)
            want, want_log = plain(logits[some], u[some], **kw)
            assert torch.equal(tokens[some], want), kw
            masses = torch.exp(logits[some].double() - logits[some].double().amax(1, keepdim=True)).sum(1)
            slack = vocab * 2.0 ** -43 / (masses if not kw else torch.ones_like(masses))
            assert ((logprobs[some].double() - want_log).abs() <= 1.1 * 2.0 ** -24 * want_log.abs() + slack).all(), kw
            few = FusedSampling.apply(logits[-2:], u[-2:], **kw)
            assert torch.equal(tokens[-2:], few[0]) and torch.equal(logprobs[-2:], few[1]), kw
        logits.fill_(1.5)  # (equal masses: exact sums)
        for kw, keep in ((dict(), vocab), (dict(top_k=4321), 4321), (dict(top_p=0.5), -(-vocab // 2)), (dict(top_k=1000), 1000)):
            tokens = FusedSampling.apply(logits, u, **kw)[0]
            assert torch.equal(tokens, torch.floor(u.double() * keep).long()), kw
    with pytest.raises(RuntimeError):
        FusedSampling.apply(torch.zeros((1, 500001), dtype=dtype, device=DEV), u[:1])
