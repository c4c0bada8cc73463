"""LogitRules on the GPU against plain operations of 64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from dimmerkv import _lib
from dimmerkv.logits import LogitRules, allow_mask
from q4_reference import rules64

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


def _first_best(x):
    best = x.amax(-1, keepdim=True)
    first = torch.where(x == best, torch.arange(x.shape[1], device=x.device), x.shape[1]).amin(-1)
    return torch.where(best[:, 0] == -float("inf"), -1, first)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab,n,n_bias,grammar", [
    (1, 1, 1, 0, False), (2, 31, 40, 3, True), (3, 1000, 200, 17, True), (5, 4097, 1, 0, False),
    (2, 20001, 500, 1024, False), (4, 131, 0, 0, True), (2, 140003, 60, 5, False)])
def test_rules_follow_the_formulas(rows, vocab, n, n_bias, grammar, dtype):
    g = torch.Generator().manual_seed(vocab)
    logits = (torch.randn(rows, vocab, generator=g) * 3).to(dtype)
    history = (torch.rand(rows, max(n, 1), generator=g).pow(2) * vocab).to(torch.int32)[:, :n]
    if n > 3:
        history[0, 1], history[0, 2] = vocab, -5  # no tokens: skipped
    lengths = [max(0, n - r) for r in range(rows)]
    prompts = [l // (r + 2) for r, l in enumerate(lengths)]
    pen = [1.0 + torch.rand(rows, generator=g), torch.rand(rows, generator=g) - 0.3, torch.rand(rows, generator=g)]
    bias = None
    if n_bias:
        ids = torch.randint(-1, vocab, (rows, n_bias), generator=g, dtype=torch.int32)
        ids[:, -1] = ids[:, 0]  # the same token twice
        bias = (ids, torch.randn(rows, n_bias, generator=g) * 2)
    allowed = None
    if grammar:
        allowed = torch.randint(-2**31, 2**31, (rows, (vocab + 31) // 32), generator=g).to(torch.int32)
        logits[rows - 1, :3] = float("nan") if vocab > 3 else 0.0
        allowed[rows - 1, 0] = allowed[rows - 1, 0] & ~7  # a NaN where the mask allows nothing
    rules = LogitRules(rows, vocab, capacity=max(n, 1) + 2, repetition=pen[0].to(DEV), frequency=pen[1], presence=pen[2],
                       bias_ids=None if bias is None else bias[0], bias_values=None if bias is None else bias[1])
    rules.load(history.to(DEV), lengths, prompts)
    mask = None if allowed is None else allowed.to(DEV)
    got, token = rules.apply(logits.to(DEV), mask)
    want = rules64(torch.nan_to_num(logits.float(), nan=0.0), history.numpy(), lengths, prompts, *(p.tolist() for p in pen),
                   None if bias is None else (bias[0].numpy(), bias[1].numpy()),
                   None if allowed is None else allowed.numpy())
    got = got.cpu().double()
    hidden = torch.isinf(want)
    assert torch.equal(torch.isinf(got), hidden)
    # Up to four roundings (quotient or product, frequency * count, two differences) and up to n_bias sums, each half
    # a float32 step of a term no larger than the sum of the absolute terms.
    size = logits.float().nan_to_num().abs().double() * 2 + 2 + n * 1.0
    if bias is not None:
        size = size + rules64(torch.zeros(rows, vocab), [[]] * rows, [0] * rows, [0] * rows, [1] * rows, [0] * rows, [0] * rows,
                              (bias[0].numpy(), bias[1].abs().numpy()))
    assert bool(((got - want).abs()[~hidden] <= (size * 2**-24 * (5 + n_bias // 8))[~hidden]).all())
    assert torch.equal(token.cpu(), _first_best(got))
    # the history is as it was; pick takes the same token into it
    assert rules.lengths.tolist() == lengths
    picked = rules.pick(logits.to(DEV), mask)
    assert torch.equal(picked.cpu(), token.cpu())
    for r in range(rows):
        t = int(token[r])
        assert int(rules.lengths[r]) == lengths[r] + (t >= 0)
        if t >= 0:
            assert int(rules.history[r, lengths[r]]) == t
    rules.check_status()


def test_long_histories_and_many_rows():
    """Counts beyond 14 bits (histories with room for more than 16383 tokens), and rows enough for the longer slices."""
    rows, vocab = 2, 140003
    g = torch.Generator(device=DEV).manual_seed(4)
    x = torch.randn(rows, vocab, generator=g, device=DEV)
    history = torch.full((rows, 20000), 5, dtype=torch.int32, device=DEV)
    history[:, :4000] = torch.randint(0, vocab, (rows, 4000), generator=g, device=DEV, dtype=torch.int32)
    rules = LogitRules(rows, vocab, capacity=20001, repetition=1.25, frequency=0.0625, presence=0.5)
    rules.load(history, prompts=[3000, 0])
    out, token = rules.apply(x)
    count = torch.zeros(rows, vocab, device=DEV)
    seen = torch.zeros(rows, vocab, dtype=torch.bool, device=DEV)
    for r, p in enumerate((3000, 0)):
        count[r] = torch.bincount(history[r, p:].long(), minlength=vocab)
        seen[r] = torch.bincount(history[r].long(), minlength=vocab) > 0
    pen = torch.full((rows, 1), 1.25, device=DEV)  # a tensor: torch divides by a number as a product with its reciprocal
    want = torch.where(seen, torch.where(x > 0, x / pen, x * pen), x)
    want = torch.where(count > 0, (want - 0.0625 * count) - 0.5, want)  # the same float32 steps: the same bits
    assert torch.equal(out, want) and torch.equal(token, _first_best(want))
    assert float(count[:, 5].min()) >= 16000
    rows = 60
    x = torch.randn(rows, vocab, generator=g, device=DEV).bfloat16()
    rules = LogitRules(rows, vocab, capacity=64, repetition=torch.linspace(1, 2, rows), presence=0.25)
    history = torch.randint(0, vocab, (rows, 50), generator=g, device=DEV, dtype=torch.int32)
    rules.load(history, prompts=[r % 50 for r in range(rows)])
    allowed = torch.randint(-2**31, 2**31, (rows, (vocab + 31) // 32), generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
    out, token = rules.apply(x, allowed)
    seen = torch.zeros(rows, vocab, dtype=torch.bool, device=DEV).scatter_(1, history.long(), True)
    made = torch.zeros(rows, vocab, dtype=torch.bool, device=DEV)
    for r in range(rows):
        made[r, history[r, r % 50:].long()] = True
    pen = torch.linspace(1, 2, rows, device=DEV)[:, None]
    want = torch.where(seen, torch.where(x > 0, x.float() / pen, x.float() * pen), x.float())
    want = torch.where(made, want - 0.25, want)
    at = torch.arange(vocab, device=DEV)
    want = torch.where((allowed[:, at // 32] >> (at % 32)) & 1 != 0, want, -float("inf"))
    assert torch.equal(out, want) and torch.equal(token, _first_best(want))
    rules.check_status()


def test_choice_at_ties_and_ends():
    x = torch.full((6, 300), -2.0, device=DEV)
    x[0, [17, 200]] = 1.5                      # equal: the lowest
    x[1, [5, 9]] = torch.tensor([-0.0, 0.0], device=DEV)
    x[2] = -float("inf")                       # nothing
    x[3, 299] = float("inf")
    x[4, [7, 250]] = float("nan")              # above all, the lowest of them
    x[5, 31] = -1.0
    rules = LogitRules(6, 300)
    out, token = rules.apply(x)
    assert token.tolist() == [17, 5, -1, 299, 7, 31]
    assert torch.equal(out.nan_to_num(nan=9.0), x.nan_to_num(nan=9.0))
    mask = allow_mask([[200], [], [3], list(range(299)), [8], [299, 298]], 300)
    assert rules.apply(x, mask)[1].tolist() == [200, -1, -1, 0, 8, 298]
    assert rules.pick(x, mask).tolist() == [200, -1, -1, 0, 8, 298]
    assert rules.lengths.tolist() == [1, 0, 0, 1, 1, 1]


def test_views_streams_graphs_and_full_histories():
    rows, vocab = 3, 1000
    g = torch.Generator(device=DEV).manual_seed(1)
    steps = [torch.randn(rows, 4, vocab + 1, generator=g, device=DEV).bfloat16() for _ in range(4)]
    def fresh():
        r = LogitRules(rows, vocab, capacity=4, repetition=1.5, frequency=0.7)
        r.load(torch.tensor([[1], [2], [3]], dtype=torch.int32))
        return r
    eager, replayed = fresh(), fresh()
    want = [eager.pick(s[:, -1, 1:]).clone() for s in steps[:3]]  # rows that start at odd addresses
    aligned = fresh()
    assert torch.equal(torch.stack([aligned.pick(s[:, -1, 1:].contiguous()) for s in steps[:3]]), torch.stack(want))
    static = steps[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fresh().pick(static[:, -1, 1:])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = replayed.pick(static[:, -1, 1:])
    for s, w in zip(steps, want):
        static.copy_(s)
        graph.replay()
        assert torch.equal(out, w)
    assert torch.equal(eager.history, replayed.history)
    replayed.check_status()
    graph.replay()  # the histories hold four tokens
    with pytest.raises(_lib.DimmerKVError, match="114"):
        replayed.check_status()
    assert torch.equal(eager.history, replayed.history)
    for bad in (static[:, -1], static[:2, -1, 1:], static[:, -1, 1:].cpu(), static[:, -1, 1:].to(torch.int32)):
        with pytest.raises(ValueError):
            eager.pick(bad)
    for mask in (torch.zeros(rows, 32, device=DEV), torch.zeros(rows, 31, dtype=torch.int32, device=DEV),
                 torch.zeros(rows, 32, dtype=torch.int32)):
        with pytest.raises(ValueError):
            eager.pick(static[:, -1, 1:], mask)
