"""Token log probabilities on the device (mi_token_logprobs via
microinfer_amd.layer.hip_logprobs) against float64 log_softmax.

Tolerances are counted in roundings of float32 (half a step is 2^-24). A log
probability is (x - M) c - log2 S: the product and c carry four roundings of
|x - M| / T, S the exp2 of each term (two) and its additions -- at most
vocab / 256 in a row, of errors that do not line up, so four times their
root -- and log2 and the last product a few of the result. The entropy is
log2 S - E / S, where E weighs exponents of up to |H| + log2 S + 10 (the
reference of the sums lies at most 2^10 below the maximum).
The order of the alternatives is exact.
"""

import math
import sys

import pytest
import torch

from microinfer_amd.layer import hip_logprobs
from microinfer_amd.layer.hip_logprobs import token_logprobs
from microinfer_amd.layer.hip_sampler import greedy_argmax
from microinfer_amd.runner import capture_graph

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF = 2.0 ** -24


def _expected(logits, temperatures):
    x = logits.double()
    if temperatures is not None:
        x = x / temperatures.double()[:, None]
    return torch.log_softmax(x, 1)


def _sums(vocab):
    return 4 * math.sqrt(vocab / 256 + 1) + 12


def _close(got, want, scale, vocab):
    """Equal infinities and NaN; else within the roundings of the docstring."""
    assert got.dtype == torch.float32
    got, want = got.double(), want.double()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isinf(), want.isinf())
    fine = want.isfinite()
    tol = HALF * (6 * scale + _sums(vocab))
    err = (got - want).abs()
    assert (err <= tol)[fine].all(), f"off by {(err - tol)[fine].max()} more than {tol.max()}"


def check(logits, tokens=None, *, top=0, temperatures=None, entropy=True):
    got = token_logprobs(logits, tokens, top=top, temperatures=temperatures, entropy=entropy)
    vocab = logits.shape[1]
    logp = _expected(logits, temperatures)
    if tokens is None:
        assert got.logprobs is None
    else:
        given = tokens.long().view(len(tokens), -1)
        inside = (given >= 0) & (given < vocab)
        want = logp.gather(1, given.clamp(0, vocab - 1))
        want = want.masked_fill(~inside, math.nan).view(tokens.shape)
        assert got.logprobs.shape == tokens.shape
        # |x - M| / T is at most |ln p| above ln p's own distance to the best.
        _close(got.logprobs, want, want.abs().nan_to_num(0, 0, 0) + 1, vocab)
    if entropy:
        p = logp.exp()
        want = -(p * logp).masked_fill(p == 0, 0).sum(1)
        weight = want.abs().nan_to_num() / math.log(2) + math.log2(vocab) + 10
        _close(got.entropy, want, weight + weight * _sums(vocab) / 6, vocab)
    else:
        assert got.entropy is None
    if top:
        order = torch.sort(logits.float(), dim=1, descending=True, stable=True).indices[:, :top]
        assert got.top_tokens.dtype == torch.int64
        assert torch.equal(got.top_tokens, order)
        want = logp.gather(1, order)
        _close(got.top_logprobs, want, want.abs().nan_to_num(0, 0, 0) + 1, vocab)
    else:
        assert got.top_tokens is None and got.top_logprobs is None
    torch.cuda.synchronize()
    assert all(int(c.abs().sum()) == 0 for c, _ in hip_logprobs._scratches.values())
    return got


def _logits(rows, vocab, dtype, seed, spread=3.0, pad=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, vocab + pad, generator=gen, device=DEV) * spread
    return x.to(dtype)[:, :vocab]


def _tokens(rows, vocab, n, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    t = torch.randint(vocab, (rows, n), generator=gen, device=DEV)
    return t[:, 0].contiguous() if n == 1 else t


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top,given,pad", [
    (1, 151936, 5, 1, 0), (64, 151936, 20, 1, 0), (600, 5000, 32, 3, 0), (7, 1, 1, 1, 0),
    (3, 2, 2, 2, 3), (5, 33, 32, 1, 0), (1, 262147, 32, 1, 0), (33, 32003, 8, 300, 5),
    (700, 4099, 1, 1, 1), (2, 40, 20, 1, 0), (1, 65536, 0, 1, 0), (513, 257, 3, 1, 7),
    (9, 2049, 31, 0, 0),
])
def test_matches_float64(dtype, rows, vocab, top, given, pad):
    logits = _logits(rows, vocab, dtype, rows + vocab, pad=pad)
    tokens = _tokens(rows, vocab, given, vocab) if given else None
    check(logits, tokens, top=top)
    check(logits, tokens, top=top, entropy=False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_temperatures(dtype):
    logits = _logits(40, 20011, dtype, 3)
    gen = torch.Generator(device=DEV).manual_seed(4)
    temperatures = 0.05 + 3 * torch.rand(40, generator=gen, device=DEV)
    temperatures[5] = 1000.0
    check(logits, _tokens(40, 20011, 1, 5), top=9, temperatures=temperatures)
    # Values that are no temperature: NaN, the order unchanged.
    bad = temperatures.clone()
    bad[:5] = torch.tensor([0.0, -1.0, math.nan, math.inf, 1e-45])
    got = token_logprobs(logits, _tokens(40, 20011, 1, 5), top=9, temperatures=bad, entropy=True)
    for x in (got.logprobs, got.entropy, got.top_logprobs.sum(1)):
        assert x[:5].isnan().all() and x[5:].isfinite().all()
    order = torch.sort(logits.float(), dim=1, descending=True, stable=True).indices[:, :9]
    assert torch.equal(got.top_tokens, order)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [151936, 3001, 70])
def test_masks_ties_and_values_out_of_order(dtype, vocab):
    low = torch.finfo(dtype).min
    rows = []

    def row(fill):
        rows.append(torch.full((vocab,), fill, device=DEV))
        return rows[-1]

    row(-math.inf)[[3, vocab - 1]] = 2.0          # two values left
    row(-math.inf)[vocab - 2] = -7.5              # one
    row(low)[[0, vocab // 2]] = 1.0               # masked with the type's lowest value
    row(low)                                      # nothing but the lowest value
    row(1.25)                                     # all equal, of both signs
    row(-1.25)
    x = row(0.0)
    x[1::2] = -0.0                                # zeros of both signs are equal
    row(0.0)[::3] = 1.0                           # many ties at the best
    row(0.0)[vocab // 2:] = 0.5                   # ties that begin in the middle
    rows.append(torch.arange(vocab, device=DEV) / vocab * 20)   # rising
    rows.append(-torch.arange(vocab, device=DEV) / vocab * 20)  # falling
    x = row(-math.inf)
    x[: vocab // 3] = 0.0                         # fewer finite at the end of the row
    x = row(low)
    x[::2] = -math.inf
    x = row(0.0)
    x[vocab // 2] = 60000.0                       # everything else vanishes
    x = row(-30.0)
    x[vocab - 5] = 40.0                           # the best far above what came before
    rows.append(torch.where(torch.arange(vocab, device=DEV) % 64 < 8, 5.0, -5.0)
                + torch.arange(vocab, device=DEV) % 7)
    logits = torch.stack([r.float() for r in rows]).to(dtype)
    tokens = torch.tensor([[0, 3, vocab - 1]], device=DEV).expand(len(rows), 3)
    for top in (1, 5, 32):
        check(logits, tokens, top=top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [151936, 9001])
def test_nan_and_infinities(dtype, vocab):
    logits = _logits(10, vocab, dtype, 8)
    logits[0, vocab - 3] = math.nan
    logits[1, 4] = math.nan
    logits[1, vocab - 1] = math.nan
    logits[2, vocab // 2] = math.inf
    logits[3] = math.nan
    logits[4] = -math.inf
    logits[5, ::2] = math.nan
    logits[6] = 1.0
    logits[6, vocab - 100] = math.nan            # ties of the first tile still come first
    logits[7] = math.inf
    logits[8, 5] = math.inf
    logits[8, 6] = math.nan
    got = check(logits, _tokens(10, vocab, 2, 1), top=32)
    assert got.logprobs[:9].isnan().all() and got.logprobs[9].isfinite().all()
    assert torch.equal(got.top_tokens[:, 0], greedy_argmax(logits))


def test_tokens_outside_the_vocabulary():
    logits = _logits(4, 1000, torch.bfloat16, 2)
    tokens = torch.tensor([[-1, 0], [1000, 999], [-(2 ** 40), 5], [2 ** 40, 7]], device=DEV)
    got = check(logits, tokens)
    assert got.logprobs[:, 0].isnan().all() and got.logprobs[:, 1].isfinite().all()
    same = token_logprobs(logits, tokens[:, 1].int())
    assert torch.equal(same.logprobs, got.logprobs[:, 1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    base = _logits(30, 4200, dtype, 6)
    for view in (base[:, :4096], base[:, 1:4100], base[::3, 3:1003], base[:, 5:6],
                 base[:5, :4000].t(), base[:1].expand(4, 4200)):
        check(view, _tokens(view.shape[0], view.shape[1], 2, 1), top=min(4, view.shape[1]))
    tokens = _tokens(30, 4200, 6, 2)[:, ::2]
    check(base, tokens, top=3, temperatures=torch.rand(60, device=DEV)[::2] + 0.1)


def test_long_rows_in_large_strides():
    # Rows more than 2^31 elements apart in one buffer.
    buffer = torch.zeros(2 ** 31 + 5000, dtype=torch.bfloat16, device=DEV)
    logits = buffer.as_strided((2, 4000), (2 ** 31 + 16, 1))
    logits.copy_(_logits(2, 4000, torch.bfloat16, 9))
    check(logits, _tokens(2, 4000, 1, 1), top=5)


def test_empty_calls():
    got = token_logprobs(torch.empty(0, 50, device=DEV),
                         torch.empty(0, dtype=torch.int64, device=DEV), top=4, entropy=True)
    assert got.logprobs.shape == (0,) and got.top_tokens.shape == (0, 4)
    assert got.entropy.shape == (0,)
    got = token_logprobs(_logits(3, 50, torch.float32, 1))
    assert got == (None, None, None, None)
    got = token_logprobs(_logits(3, 50, torch.float32, 1),
                         torch.empty(3, 0, dtype=torch.int64, device=DEV))
    assert got.logprobs.shape == (3, 0)


def test_calls_are_repeatable_bit_for_bit():
    logits = _logits(16, 151936, torch.bfloat16, 12)
    tokens = _tokens(16, 151936, 1, 3)
    first = token_logprobs(logits, tokens, top=20, entropy=True)
    for _ in range(5):
        again = token_logprobs(logits, tokens, top=20, entropy=True)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_two_graphs_and_eager_calls_share_nothing():
    rows, vocab = 8, 151936
    inputs = [_logits(rows, vocab, torch.bfloat16, 20 + i) for i in range(2)]
    tokens = _tokens(rows, vocab, 1, 5)
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for x in inputs:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            token_logprobs(x, tokens, top=7, entropy=True)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with capture_graph(graph, stream=side):
            outs.append(token_logprobs(x, tokens, top=7, entropy=True))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for replay in range(4):
        for i, x in enumerate(inputs):
            x.copy_(_logits(rows, vocab, torch.bfloat16, 100 + 2 * replay + i))
        want = [token_logprobs(x, tokens, top=7, entropy=True) for x in inputs]
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):  # side by side
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(side):
            beside = token_logprobs(inputs[0], tokens, top=7, entropy=True)
        torch.cuda.synchronize()
        for out, expect in zip(outs + [beside], want + want[:1]):
            assert all(torch.equal(a, b) for a, b in zip(out, expect)), f"replay {replay}"


def _rows_that_turn_late(vocab, dtype):
    """Rows whose later tiles overthrow what the first showed (a tile is 8192
    values in 16 bits, 4096 in 32)."""
    at = torch.arange(vocab, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(11)
    noise = 2.5 * torch.randn(vocab, generator=gen, device=DEV)
    few = at % 64 < 8
    rows = [
        torch.where(at < 8192, -math.inf, noise),           # the first tile masked
        torch.where(at < 8192, torch.finfo(dtype).min, noise),
        torch.where(at < vocab - 20, -math.inf, noise),     # all but the last values masked
        noise + at // 4096 * 14.0,                          # the reference moves every tile
        noise + at // 2000 * 3.0,
        at / vocab * 60 - 30,                               # rising, falling
        30 - at / vocab * 60,
        torch.where(at < 8192, noise - 20, 5.0),            # thousands of equal best ones, late
        torch.where(at >= vocab // 2, 3.0, noise.clamp(max=3.0)),
        torch.where(few & (at > 9000), 20.0 + at % 7, noise),   # many large ones in few lanes
        torch.where(few & (at > 9000), 20.0 + at / vocab, noise),
        torch.where(at % 4096 < 5, 10.0, -10.0),            # ties over all tiles
        torch.where(at < 9000, -0.0, 0.0),
        torch.where(at == 3, 60.0, noise - 40),             # everything vanishes behind it
        torch.where(at == vocab - 2, 60.0, noise),
        torch.where(at > vocab - 3000, math.nan, noise),    # more NaN than a list holds
        torch.where(at == vocab - 9, math.nan, noise + at // 4096 * 14.0),
        torch.where(at == vocab - 9, math.inf, noise),
        torch.where(at % 3 == 0, -math.inf, noise),
        noise,
    ]
    return torch.stack([r.float() for r in rows]).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(1040, 50021), (300, 151936), (1040, 151936)])
def test_rows_that_turn_late(dtype, rows, vocab, monkeypatch):
    # 1040 rows are one part each, of 7 to 38 tiles; 300 are a few parts of
    # several tiles. The type's lowest value at a temperature of 0.3 has a log
    # probability of -1.1e39, which is -inf in float32.
    def expected(logits, temperatures, exact=_expected):
        want = exact(logits, temperatures)
        return want.masked_fill(want < torch.finfo(torch.float32).min, -math.inf)

    monkeypatch.setattr(sys.modules[__name__], "_expected", expected)
    kinds = _rows_that_turn_late(vocab, dtype)
    n = len(kinds)
    logits = kinds.repeat(rows // n, 1)
    assert len(logits) == rows
    tokens = torch.tensor([[0, 3, vocab - 1, vocab // 2]], device=DEV).expand(rows, 4)
    hot = (torch.arange(rows, device=DEV) // n % 3 == 2).float() * 1.7 + 0.3
    for top in (1, 5, 32):
        got = check(logits, tokens, top=top, temperatures=hot if top == 5 else None)
        again = got.top_tokens.view(rows // n, n, top)
        assert bool((again == again[:1]).all())
    check(logits, tokens)


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_least_temperature(dtype):
    # The smallest normal float32 and from there on; below it, NaN.
    least = torch.finfo(torch.float32).tiny
    logits = _logits(7, 9001, dtype, 13)
    logits[:, 77] = 31.0
    logits[1:, 5000] = 31.0
    values = [least, least, 2 * least, 1e-30, least / 2, 4.3e-39, 1e-45]
    temperatures = torch.tensor(values, device=DEV)
    got = token_logprobs(logits, torch.full((7,), 77, device=DEV), top=4, entropy=True,
                         temperatures=temperatures)
    fine = [0.0] + [-math.log(2)] * 3  # the best alone, or both of them
    want = torch.tensor(fine + [math.nan] * 3, device=DEV, dtype=torch.float64)
    assert torch.allclose(got.logprobs.double(), want, rtol=2 ** -22, atol=0, equal_nan=True)
    assert torch.allclose(got.entropy.double(), -want, rtol=2 ** -22, atol=0, equal_nan=True)
    # Differences of 10 and more: past float32's range below 1e-37, not at 1e-30.
    assert bool((got.top_logprobs[:3, 2:] == -math.inf).all())
    assert bool((got.top_logprobs[3, 2:] < -1e30).all())
    assert bool(got.top_logprobs[4:].isnan().all())
    order = torch.sort(logits.float(), dim=1, descending=True, stable=True).indices[:, :4]
    assert torch.equal(got.top_tokens, order)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_part_without_values(dtype):
    # Parts leave room for rows that start off the 16-byte grid: aligned rows of
    # whole tiles leave the last one empty.
    for rows, vocab in ((4, 32768), (3, 8192), (1, 262144)):
        logits = _logits(rows, vocab, dtype, vocab)
        check(logits, _tokens(rows, vocab, 1, 2), top=32)
        check(logits, top=0)
        logits[0] = -math.inf
        check(logits, _tokens(rows, vocab, 1, 2), top=3)
