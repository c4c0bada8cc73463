"""The paged 4-bit cache and the logit rules at their edges: cells without a spread, masks, empty calls, captured steps,
and what the drivers do when something has failed."""

from __future__ import annotations

import pytest
import torch

import tinymodel as tm
from dimmerkv import _lib, dimmer
from dimmerkv.compressed_attention import greedy_answer, greedy_decode_batch
from dimmerkv.logits import LogitRules
from dimmerkv.q4 import Q4Batch, Q4Context, restore
from test_gpu_q4 import _check, _filled, _rows, _Tokens
from test_gpu_rules import _first_best

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


@pytest.mark.parametrize("q_len", [1, 5, 12, 90])
@pytest.mark.parametrize("dim", [64, 128])
def test_groups_whose_least_value_rounds_above_their_largest(dim, q_len):
    """bfloat16 groups of next to nothing: low, rounded to float16, lies above every element. Their scale is +0, held
    and new tokens alike, and the tokens beside them come out as ever."""
    held, counts, dtype = [130, 64], [q_len, q_len], torch.bfloat16
    batch, query, _, _, keys, values = _filled(2, 4, 2, dim, dtype, held, counts, q_len, seed=31)
    batch.trim([0, 0])
    values[:, :, 3::7, :64] = -1e-8
    values[:, :, 5::11] = -1.5e-6
    values[0, :, held[0]] = -1.5e-6  # the first new token of one conversation
    keys[:, :, 2::9, :64] = -1.5e-6
    batch.plan(held, held[0])
    batch.append(0, keys[:, :, :held[0]], values[:, :, :held[0]])
    batch.plan(counts, q_len)
    new = [torch.stack([x[s, :, h:h + q_len] for s, h in enumerate(held)]) for x in (keys, values)]
    out = batch.attend_layer(0, query, *new, dim ** -0.5)
    _check(out, query, keys, values, held, counts, dim ** -0.5)
    heads = batch.cells[0, :, :, 64 * dim:].reshape(batch.table.n_pages, 2, 64, -1, 2, 2)  # token, group, (scale, low), bytes
    slots = batch.table.slots(sum(held[:1]) + q_len)[0].long()
    high = heads[slots // 64, :, slots % 64, :, 0, 1]
    assert int(high.max()) < 128  # no sign
    batch.check_status()


@pytest.mark.parametrize("rows,vocab", [(600, 40000), (40, 1000)])
def test_a_full_history_leaves_the_other_rows_whole(rows, vocab):
    """A row with no room tells; another row of the call has its own best token, or, where it began after that, none:
    never the best of a part of the vocabulary, and never one that its history does not have."""
    g = torch.Generator(device=DEV).manual_seed(7)
    x = torch.randn(rows, vocab, generator=g, device=DEV)
    best = x.argmax(-1)
    for _ in range(30):
        rules = LogitRules(rows, vocab, capacity=4)
        rules.lengths[0] = 4
        token = rules.pick(x)
        with pytest.raises(_lib.DimmerKVError, match="114"):
            rules.check_status()
        assert int(token[0]) in (-1, int(best[0])) and int(rules.lengths[0]) == 4
        made = token >= 0
        assert torch.equal(token[made], best[made])
        assert torch.equal(rules.lengths[1:], made[1:].int())
        assert torch.equal(rules.history[1:, 0].long(), token[1:])  # -1 where nothing was appended


def _prefilled(model, rows, max_tokens=128):
    batch = Q4Batch(rows, layers=2, kv_heads=8, q_heads=32, head_dim=64, max_tokens=max_tokens, dtype=model.dtype)
    ids = tm.context_ids().to(DEV)[0, :rows * 40].view(rows, 40)
    dimmer.STATE.compressed = batch
    try:
        model(input_ids=ids, past_key_values=batch.cache, position_ids=torch.arange(40, device=DEV)[None].expand(rows, -1),
              use_cache=True)
    finally:
        dimmer.STATE.compressed = None
    return batch


def test_the_batch_driver_tells_a_full_history_at_its_last_step():
    model = tm.build_model(torch.bfloat16, DEV)
    dimmer.install(model)
    with torch.inference_mode():
        for steps, full in ((3, False), (4, True)):
            rules = LogitRules(2, 1024, capacity=3)
            args = (torch.tensor([[1], [2]]), torch.full((2, 1), 40), steps)
            batch = _prefilled(model, 2)
            if full:
                with pytest.raises(_lib.DimmerKVError, match="114"):
                    greedy_decode_batch(model, batch, batch.cache, *args, rules=rules)
            else:
                out, moved = greedy_decode_batch(model, batch, batch.cache, *args, rules=rules)
                assert torch.equal(rules.history.cpu(), out.int())
                assert moved["d2h_bytes_per_step"] == 2 * 8 + 4 + 4  # the ids and two status words


def test_an_answer_over_a_context_without_room_is_no_answer():
    """Tokens beyond a context's room, or values that no cell holds, end greedy_answer with the error."""
    model = tm.build_model(torch.bfloat16, DEV)
    dimmer.install(model)
    question = tm.question_ids().to(DEV)[None]
    with torch.inference_mode():
        # two pages hold 128 tokens; a question of 8 and three of four answered tokens are stored
        for tokens, room, fits in ((117, 11, True), (118, 10, False), (121, 7, False)):
            cache, _ = dimmer.prefill_with_scores(model, tm.context_ids().to(DEV)[:, :tokens])
            keys, values = [l.keys for l in cache.layers], [l.values for l in cache.layers]
            context = Q4Context(keys, values, model, dtype=torch.bfloat16, room=room)
            args = (model, _Tokens(), context, context.exact_cache, question, tokens, 4)
            if fits:
                assert len(greedy_answer(*args)[0].split()) == 4
                context.check_status()
            else:
                with pytest.raises(_lib.DimmerKVError, match="9112"):
                    greedy_answer(*args)
        values[1][0, 3, 17, 5] = float("inf")
        context = Q4Context(keys, values, model, dtype=torch.bfloat16)
        with pytest.raises(_lib.DimmerKVError, match="8113"):
            greedy_answer(model, _Tokens(), context, context.exact_cache, question, tokens)
    assert dimmer.STATE.compressed is None


class _Layer:
    layer_idx = 0


def test_masks_that_hide_what_the_attention_sees_are_told():
    """A mask of more columns than new tokens has to show every older one, for each of its heads; of rows that bring
    fewer tokens only the real ones count."""
    batch = Q4Batch(2, layers=1, kv_heads=2, q_heads=4, head_dim=64, max_tokens=200)
    k, v, q = (_rows(2, h, 3, 64, torch.bfloat16, 5 + h) for h in (2, 2, 4))
    order = torch.ones(3, 3, dtype=torch.bool, device=DEV).tril()
    low = torch.finfo(torch.bfloat16).min

    def told(mask, counts=None):
        batch.begin(counts)
        batch.attend(_Layer, q, k, v, mask, 0.125)
        code = int(batch.status)
        batch.reset_status()
        return code

    def wide(old, heads=1, rows=2):
        return torch.cat([torch.ones(rows, heads, 3, old, dtype=torch.bool, device=DEV),
                          order.expand(rows, heads, 3, 3)], -1)

    additive = lambda m: torch.zeros(m.shape, dtype=torch.bfloat16, device=DEV).masked_fill_(~m, low)
    for old, heads, rows in ((0, 1, 2), (3, 1, 2), (6, 4, 1), (9, 4, 2)):
        m = wide(old, heads, rows)
        assert told(m) == 0 and told(additive(m)) == 0
    hidden = wide(12)
    hidden[1, 0, 2, 4] = False                       # an older token
    assert told(hidden) == 115 and told(additive(hidden)) == 115
    assert told(hidden, [3, 2]) == 0                 # its row is padding
    assert told(hidden, [3, 3]) == 115
    head = wide(15, heads=4)
    head[0, 3, 1, 0] = False                         # of the last head alone
    assert told(head) == 115
    head = wide(0, heads=4)
    head[0, 1, 0, 2] = True                          # shows a later token, in one head
    assert told(head) == 115
    for bad in (wide(0)[:, 0], wide(0)[..., :2]):
        with pytest.raises(ValueError):
            batch.attend(_Layer, q, k, v, bad, 0.125)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_calls_without_a_token(dtype):
    batch = Q4Batch(2, layers=1, kv_heads=2, q_heads=4, head_dim=64, max_tokens=64, dtype=dtype)
    batch.plan([3, 5], 5)
    k, v = _rows(2, 2, 5, 64, dtype, 1), _rows(2, 2, 5, 64, dtype, 2)
    batch.append(0, k, v)
    first = batch._slots
    want = batch.read(0)
    none = torch.zeros(2, 2, 0, 64, dtype=dtype, device=DEV)
    for counts in (None, [0, 0]):
        assert batch.plan(counts, 0).shape == (2, 0)
        batch.append(0, none, none)
        assert [x.shape for x in batch.read(0)] == [none.shape] * 2
        query = torch.zeros(2, 4, 0, 64, dtype=dtype, device=DEV)
        for key in (none, None):
            assert batch.attend_layer(0, query, key, key, 0.125).shape == (2, 0, 4, 64)
    assert batch.lengths.tolist() == [3, 5]
    assert all(torch.equal(a, b) for a, b in zip(batch.read(0, first), want))
    keys, values = restore([none[:1]] * 2, [none[:1]] * 2)
    assert [x.shape for x in keys + values] == [(1, 2, 0, 64)] * 4
    batch.check_status()


def test_captured_steps_grow_over_the_whole_gpu():
    """A step captured on an empty batch and replayed until it is long: the work is split as for the lengths that replays
    reach, by the replays and by eager calls behind them, so that the results are an eager batch's."""
    dim, kv, hq, n = 64, 2, 8, 512
    batches = [Q4Batch(1, layers=1, kv_heads=kv, q_heads=hq, head_dim=dim, max_tokens=16000) for _ in range(2)]
    k, v = _rows(1, kv, n, dim, torch.bfloat16, 3, "key"), _rows(1, kv, n, dim, torch.bfloat16, 4)
    one = [_rows(1, h, 1, dim, torch.bfloat16, 5 + i) for i, h in enumerate((hq, kv, kv))]
    captured, eager = batches
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.plan(None, n)
        captured.append(0, k, v)
        captured.plan()
        out = captured.attend_layer(0, *one, 0.125)
    for _ in range(20):
        graph.replay()
        eager.plan(None, n)
        eager.append(0, k, v)
        eager.plan()
        want = eager.attend_layer(0, *one, 0.125)
        assert torch.equal(out, want)
    assert captured.lengths.tolist() == eager.lengths.tolist() == [20 * (n + 1)]
    for batch in batches:
        batch.plan()
    assert torch.equal(captured.attend_layer(0, *one, 0.125), eager.attend_layer(0, *one, 0.125))
    assert captured.table.bound >= int(captured.lengths)
    captured.check_status()


@pytest.mark.parametrize("q_len", [1, 4, 40])
def test_a_plan_that_failed_stores_nothing(q_len):
    """Attention with the slots of a failed plan, once the status word is cleared: the cells stay as they were, in the
    form that stores the tokens itself as in the other."""
    batch = Q4Batch(1, layers=1, kv_heads=2, q_heads=4, head_dim=64, max_tokens=128)
    k, v, q = (_rows(1, h, q_len, 64, torch.bfloat16, i) for i, h in ((1, 2), (2, 2), (3, 4)))
    held = 128 - q_len
    batch.plan([held], held)
    batch.append(0, *(_rows(1, 2, held, 64, torch.bfloat16, i) for i in (5, 6)))
    batch.plan(None, q_len)
    batch.attend_layer(0, q, k, v, 0.125)
    slots = batch.table.slots(128)
    want = batch.read(0, slots)
    assert bool((batch.plan(None, q_len) == -1).all())
    with pytest.raises(_lib.DimmerKVError, match="9112"):
        batch.check_status()
    batch.reset_status()
    batch.attend_layer(0, q, 2 * k, 2 * v, 0.125)
    assert all(torch.equal(a, b) for a, b in zip(batch.read(0, slots), want))
    batch.check_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,q_len", [(64, 3), (128, 40), (64, 90), (128, 150)])
def test_attention_of_other_strides_signs_and_rows(dim, q_len, dtype):
    """Both forms over tensors at odd offsets and strides, under a negative scaling, and with a row that is not finite."""
    held, counts = [200, 0, 65], [q_len, q_len - 1, 1]
    batch, query, k, v, keys, values = _filled(3, 8, 2, dim, dtype, held, counts, q_len, seed=41)
    want = batch.attend_layer(0, query, k, v, 0.1)
    _check(want, query, keys, values, held, counts, 0.1)
    flat = torch.zeros(query.numel() + 3, dtype=dtype, device=DEV)
    odd = flat[3:].view(3, q_len, 8, dim).transpose(1, 2)
    odd.copy_(query)
    wide = torch.zeros(3, 2, q_len, dim + 4, dtype=dtype, device=DEV)
    wide[..., :dim] = k
    backwards = v.flip(3).contiguous().flip(3)
    assert torch.equal(batch.attend_layer(0, odd, wide[..., :dim], backwards, 0.1), want)
    heads_last = query.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)  # no dense last dimension
    assert torch.equal(batch.attend_layer(0, heads_last, None, None, 0.1), want)
    # a scaling below zero is the same as negated queries
    negative = batch.attend_layer(0, query, None, None, -0.1)
    _check(negative, -query, keys, values, held, counts, 0.1)
    # one row that is not finite: the others as they were
    for bad in (float("nan"), float("inf")):
        spoilt = query.clone()
        spoilt[0, 5, 1, 7] = bad
        out = batch.attend_layer(0, spoilt, None, None, 0.1)
        assert bad == bad or bool(out[0, 1, 5].isnan().all())
        out[0, 1, 5] = want[0, 1, 5]
        assert torch.equal(out, want)
    batch.check_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_batch_driver_picks_the_formulas_tokens(dtype):
    """greedy_decode_batch under penalties: every token is the best of the rules' formulas on the logits of its step,
    made by the same model over a second batch with the same rows."""
    model = tm.build_model(dtype, DEV)
    dimmer.install(model)
    rows, steps = 3, 7
    with torch.inference_mode():
        start, pos = torch.tensor([[4], [5], [6]]), torch.full((rows, 1), 40)
        rules = LogitRules(rows, 1024, capacity=64, repetition=1.5, frequency=0.25, presence=0.125)
        prompts = tm.context_ids().to(DEV)[0, :rows * 40].view(rows, 40)
        rules.load(prompts)
        batch = _prefilled(model, rows)
        out, _ = greedy_decode_batch(model, batch, batch.cache, start, pos, steps, rules=rules)
        again = _prefilled(model, rows)
        dimmer.STATE.compressed = again
        try:
            ids = start.to(DEV)
            for i in range(steps):
                x = model(input_ids=ids, past_key_values=again.cache, position_ids=pos.to(DEV) + i, use_cache=True).logits
                x = x[:, -1].float()
                made = torch.zeros(rows, 1024, device=DEV)
                if i:
                    made.scatter_add_(1, out[:, :i].to(DEV), torch.ones(rows, i, device=DEV))
                seen = made.scatter(1, prompts, 1.0) > 0
                x = torch.where(seen, torch.where(x > 0, x / torch.full_like(x, 1.5), x * 1.5), x)
                x = torch.where(made > 0, x - 0.25 * made - 0.125, x)
                assert torch.equal(_first_best(x).cpu(), out[:, i])
                ids = out[:, i:i + 1].to(DEV)
        finally:
            dimmer.STATE.compressed = None
    assert rules.lengths.tolist() == [40 + steps] * rows
    assert torch.equal(rules.history[:, 40:40 + steps].cpu().long(), out)


def test_a_pass_that_is_refused_plans_nothing():
    """The hook looks at a pass's tensors before it makes room for their tokens."""
    batch = Q4Batch(2, layers=1, kv_heads=2, q_heads=4, head_dim=64, max_tokens=64)
    q, k = _rows(2, 4, 3, 64, torch.bfloat16, 1), _rows(2, 2, 3, 64, torch.bfloat16, 2)
    batch.begin([3, 1])
    for query, key, value in ((q[:1], k[:1], k[:1]), (q, k[:, :1], k[:, :1]), (q[:, :2], k, k), (q, k, k[..., :32]), (q, k.cpu(), k),
                              (q, k, k[:, :, :2])):
        with pytest.raises(ValueError):
            batch.attend(_Layer, query, key, value, None, 0.125)
        assert batch.lengths.tolist() == [0, 0]
    order = torch.ones(2, 1, 3, 3, dtype=torch.bool, device=DEV).tril()
    for mask in (order[:, :, :2], order[..., :2], order[0], order.cpu(), order.repeat(2, 1, 1, 1)[:3]):
        with pytest.raises(ValueError):
            batch.attend(_Layer, q, k, k, mask, 0.125)
        assert batch.lengths.tolist() == [0, 0]
    out, _ = batch.attend(_Layer, q, k, k, order, 0.125)
    assert batch.lengths.tolist() == [3, 1] and not out[1, 1:].any()  # the counts of begin still held
    batch.check_status()
