"""The paged 4-bit cache on the GPU against plain implementations: tables, cells, attention, and a decode of a model
over them."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import tinymodel as tm
from dimmerkv import _lib, dimmer
from dimmerkv.compressed_attention import greedy_answer, greedy_decode_batch
from dimmerkv.logits import LogitRules, allow_mask
from dimmerkv.methods import Methods
from dimmerkv.paging import PageTable
from dimmerkv.q4 import Q4Batch, Q4Context, dequantise4, quantise4
from q4_reference import PlainTable, attend64, attend_tolerance, cells64

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


# ------------------------------------------------------------------------------------------------ tables
def _same(table, plain):
    n = int(table.n_free)
    assert table.free[:n].tolist() == plain.free
    assert np.array_equal(table.blocks.cpu().numpy(), plain.array())
    assert table.lengths.tolist() == plain.lengths and table.starts.tolist() == plain.starts


@pytest.mark.parametrize("n_seq,q_len", [(1, 1), (3, 65), (40, 7), (1500, 3), (5, 4000)])
def test_tables_follow_the_plain_ones(n_seq, q_len):
    rng = np.random.default_rng(n_seq)
    cap = 2 * q_len + 130
    table, plain = PageTable(n_seq, n_seq * 70 + 200, cap), PlainTable(n_seq, n_seq * 70 + 200, cap)
    for step in range(6):
        if step in (2, 4):
            keep = [int(k) for k in rng.integers(0, q_len + 70, n_seq)]
            keep[0] = 0
            table.trim(torch.tensor(keep, dtype=torch.int32, device=DEV))
            plain.trim(keep)
            _same(table, plain)
        counts = [int(c) for c in rng.integers(0, q_len + 1, n_seq)]
        counts = [min(c, cap - l) for c, l in zip(counts, plain.lengths)]
        slots = table.plan(counts, q_len)
        want = plain.plan(counts, q_len)
        assert np.array_equal(slots.cpu().numpy(), want)
        _same(table, plain)
    full = table.slots(cap).cpu().numpy()
    for s in range(n_seq):
        n = plain.lengths[s]
        assert (full[s, n:] == -1).all()
        assert full[s, :n].tolist() == [plain.blocks[s][i // 64] * 64 + i % 64 for i in range(n)]
    table.trim(table.starts)  # a count vector that the kernel changes
    plain.trim(list(plain.starts))
    _same(table, plain)
    table.check_status()


def test_a_plan_that_fails_changes_nothing():
    def state(t):
        return [x.clone() for x in (t.blocks, t.lengths, t.starts, t.free, t.n_free)]

    table = PageTable(3, 4, 192)
    table.plan([64, 1, 0], 64)
    before = state(table)
    for counts, q_len, code in (([1, 64, 65], 65, 111), ([129, 0, 0], 129, 112), ([2, 0, 0], 1, 112), ([-1, 0, 0], 1, 112)):
        slots = table.plan(counts, q_len)
        assert bool((slots == -1).all())
        for a, b in zip(state(table), before):
            assert torch.equal(a, b)
        with pytest.raises(_lib.DimmerKVError) as e:
            table.check_status()
        assert str(9000 + code) in str(e.value)
        # inert until it is reset
        assert bool((table.plan([1, 1, 1], 1) == -1).all()) and torch.equal(table.lengths, before[1])
        assert bool((table.slots(8) == -1).all())
        table.reset_status()
    table.trim([0, -1, 0])
    with pytest.raises(_lib.DimmerKVError):
        table.check_status()
    table.reset_status()
    for a, b in zip(state(table), before):
        assert torch.equal(a, b)
    table.plan([0, 63, 128], 128)  # exactly the pages that are left
    table.check_status()
    assert int(table.n_free) == 0


def test_tables_refuse_wrong_counts():
    table = PageTable(2, 4, 64)
    for counts in ([1], torch.ones(2, dtype=torch.int64, device=DEV), torch.ones(2, dtype=torch.int32),
                   torch.ones(3, dtype=torch.int32, device=DEV)):
        with pytest.raises(ValueError):
            table.plan(counts, 1)
    with pytest.raises(ValueError):
        table.plan(None, -1)
    with pytest.raises(ValueError):
        table.slots(65)


# ------------------------------------------------------------------------------------------------ cells
def _rows(n, heads, tokens, dim, dtype, seed, kind="value"):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(n, tokens, heads, dim, generator=g, device=DEV)
    if kind == "key":
        c = torch.arange(dim, device=DEV)
        x = x * (0.6 + 2.0 * (c % 29 == 3)) + torch.sin(c * 1.7) * 1.5
    return x.to(dtype).transpose(1, 2)  # the strides that a projection leaves


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,heads,n,q_len", [(64, 2, 1, 1), (128, 8, 3, 67), (64, 3, 5, 130), (128, 1, 2, 64)])
def test_cells_hold_what_the_definition_says(dim, heads, n, q_len, dtype):
    batch = Q4Batch(n, layers=2, kv_heads=heads, q_heads=heads, head_dim=dim, max_tokens=q_len + 9, dtype=dtype)
    batch.plan([7] + [5] * (n - 1), 9)  # the rows below start inside a page
    k0, v0 = (_rows(n, heads, 9, dim, dtype, s) for s in (8, 9))
    for layer in range(2):
        batch.append(layer, k0, v0)
    counts = [max(0, q_len - 3 * s) for s in range(n)]
    first = batch._slots
    batch.plan(counts, q_len)
    k, v = _rows(n, heads, q_len, dim, dtype, 1, "key"), _rows(n, heads, q_len, dim, dtype, 2)
    k[:, 0, 0, :4] = 0.0
    v[0, 0, 0] = -3.0                                # constant groups
    k[0, 0, 0, 0], k[0, 0, 0, 1] = 32768.0, -32768.0  # the largest that a cell holds
    pad = torch.arange(q_len, device=DEV) >= torch.tensor(counts, device=DEV)[:, None]
    k.masked_fill_(pad[:, None, :, None], float("nan"))  # behind the counts: never read
    v.masked_fill_(pad[:, None, :, None], float("inf"))
    batch.append(1, k, v)
    got = batch.read(1)
    for x, y in zip((k, v), got):
        # The float32 value is the exact one to 2^-24, and rounds to the 16-bit neighbour of it: equal, or one
        # 16-bit step apart where the exact value lies within that of a border.
        want = torch.where(pad[:, None, :, None], 0.0, torch.nan_to_num(cells64(x)[0], nan=0.0))
        assert bool(((y.double() - want).abs() <= want.abs() * (torch.finfo(dtype).eps / 2 + 2**-23) + 1e-7).all())
        codes = quantise4(torch.where(pad[:, None, :, None], 0.0, x.float()))
        assert torch.equal(y, torch.where(pad[:, None, :, None], 0.0, dequantise4(*codes)).to(dtype))
    # what was there stays, in this layer and in the other
    for layer in range(2):
        a, b = batch.read(layer, first)
        for x, y in zip((k0, v0), (a, b)):
            for s, c in enumerate([7] + [5] * (n - 1)):
                assert torch.equal(y[s, :, :c], dequantise4(*quantise4(x[s, :, :c])).to(dtype))
                assert not y[s, :, c:].any()
    batch.check_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,q_len", [(64, 5201), (128, 2601)])
def test_cells_of_long_prompts(dim, q_len, dtype):
    """More rows than the GPU takes at once, for which a lane has more of a row."""
    batch = Q4Batch(2, layers=1, kv_heads=8, q_heads=8, head_dim=dim, max_tokens=q_len + 3, dtype=dtype)
    batch.plan([3, 0], 3)  # one starts inside a page, at an odd token
    few = [_rows(2, 8, 3, dim, dtype, s) for s in (8, 9)]
    batch.append(0, *few)
    first = batch._slots
    counts = torch.tensor([q_len, q_len - 334], device=DEV)
    batch.plan(counts.tolist(), q_len)
    k, v = _rows(2, 8, q_len, dim, dtype, 1, "key"), _rows(2, 8, q_len, dim, dtype, 2)
    pad = (torch.arange(q_len, device=DEV) >= counts[:, None])[:, None, :, None]
    k.masked_fill_(pad, float("nan"))
    v.masked_fill_(pad, float("inf"))
    batch.append(0, k, v)
    for x, y in zip((k, v), batch.read(0)):
        want = dequantise4(*quantise4(torch.where(pad, 0.0, x.float())))
        assert torch.equal(y, torch.where(pad, 0.0, want).to(dtype))
    for x, y in zip(few, batch.read(0, first)):
        assert torch.equal(y[0], dequantise4(*quantise4(x[0])).to(dtype))
    batch.check_status()


def test_codes_at_the_borders_between_two():
    """x exactly half way between two codes goes to the even one, one 16-bit step beside it to its own side."""
    dim = 64
    x = torch.zeros(1, 1, 3, dim, dtype=torch.float16, device=DEV)
    half = (torch.arange(15, device=DEV) + 0.5).half()
    x[..., 15] = 15.0                                   # scale 1, low 0
    x[0, 0, 0, 16:31] = half
    x[0, 0, 1, 16:31] = torch.nextafter(half, torch.full_like(half, 100))
    x[0, 0, 2, 16:31] = torch.nextafter(half, torch.zeros_like(half))
    batch = Q4Batch(1, layers=1, kv_heads=1, q_heads=1, head_dim=dim, max_tokens=3, dtype=torch.float16)
    batch.plan(None, 3)
    batch.append(0, x, x)
    k, v = batch.read(0)
    assert torch.equal(k, v) and torch.equal(k.double(), cells64(x)[0])
    assert k[0, 0, 0, 16:31].tolist() == [0, 2, 2, 4, 4, 6, 6, 8, 8, 10, 10, 12, 12, 14, 14]
    assert k[0, 0, 1, 16:31].tolist() == list(range(1, 16)) and k[0, 0, 2, 16:31].tolist() == list(range(15))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 40000.0])
def test_values_without_a_cell_are_told(bad):
    batch = Q4Batch(1, layers=1, kv_heads=2, q_heads=2, head_dim=64, max_tokens=64)
    batch.plan(None, 2)
    k = torch.ones(1, 2, 2, 64, dtype=torch.bfloat16, device=DEV)
    v = k.clone()
    v[0, 1, 1, 63] = bad
    batch.append(0, k, v)
    with pytest.raises(_lib.DimmerKVError, match="8113"):
        batch.check_status()
    assert not any(x.any() for x in batch.read(0))  # inert
    batch.reset_status()
    batch.append(0, k, k)
    batch.check_status()


def test_batch_refuses_wrong_tensors():
    batch = Q4Batch(2, layers=1, kv_heads=2, q_heads=4, head_dim=64, max_tokens=64)
    k = torch.zeros(2, 2, 1, 64, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16, device=DEV)
    for call in (lambda: batch.append(0, k, k), lambda: batch.read(0), lambda: batch.attend_layer(0, q, k, k, 1.0)):
        with pytest.raises(RuntimeError):
            call()
    batch.plan()
    for call in (lambda: batch.append(1, k, k), lambda: batch.append(0, k[:, :1], k), lambda: batch.append(0, k.cpu(), k),
                 lambda: batch.attend_layer(0, q[:, :3], k, k, 1.0), lambda: batch.attend_layer(0, q, k, None, 1.0),
                 lambda: batch.attend_layer(0, q, k, k, 1.0, out_dtype=torch.float16),
                 lambda: batch.read(0, torch.zeros(2, 3, device=DEV)),
                 lambda: batch.read(0, torch.zeros(3, 3, dtype=torch.int32, device=DEV))):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------------------------------------ attention
def _filled(n, q_heads, kv_heads, dim, dtype, held, counts, q_len, seed=0, chunk=1000):
    """A batch that holds ``held`` tokens and has ``counts`` more planned, with every key and value of it."""
    total = max(h + c for h, c in zip(held, counts))
    batch = Q4Batch(n, layers=1, kv_heads=kv_heads, q_heads=q_heads, head_dim=dim, max_tokens=max(1, total) + 70, dtype=dtype)
    batch.cells.fill_(0xff)  # NaN headers wherever nothing was stored
    keys, values = _rows(n, kv_heads, total, dim, dtype, seed, "key"), _rows(n, kv_heads, total, dim, dtype, seed + 1)
    for first in range(0, max(held), chunk):
        part = [min(chunk, max(0, h - first)) for h in held]
        size = max(part)
        batch.plan(part, size)
        batch.append(0, keys[:, :, first:first + size], values[:, :, first:first + size])
    batch.plan(counts, q_len)
    query = _rows(n, q_heads, q_len, dim, dtype, seed + 2)
    new = [torch.zeros(n, kv_heads, q_len, dim, dtype=dtype, device=DEV) for _ in range(2)]
    for s in range(n):
        for x, y in zip(new, (keys, values)):
            x[s, :, :counts[s]] = y[s, :, held[s]:held[s] + counts[s]]
    return batch, query, new[0], new[1], keys, values


def _check(out, query, keys, values, held, counts, scaling):
    rows = query.shape[1] // keys.shape[1] * query.shape[2]
    for s, (h, c) in enumerate(zip(held, counts)):
        assert not out[s, c:].any()
        if c:
            want, parts = attend64(query[s, :, :c], keys[s, :, :h + c], values[s, :, :h + c], h, scaling)
            err = (out[s, :c].double() - want).abs() - attend_tolerance(want, parts, query.dtype, out.dtype, rows)
            assert float(err.max()) <= 0, (s, float(err.max()))


CASES = [
    # q_heads, kv_heads, dim, held, counts, q_len
    (4, 1, 64, [0], [1], 1),
    (24, 8, 128, [1], [1], 1),
    (24, 8, 128, [63, 64, 65, 0, 200], [1, 1, 1, 0, 1], 1),
    (32, 8, 64, [127, 16, 1000], [1, 1, 1], 1),
    (32, 8, 64, [700, 0, 5, 63], [3, 5, 0, 2], 5),
    (24, 8, 128, [129, 300], [4, 1], 4),
    (8, 8, 128, [500], [1], 1),
    (7, 1, 64, [333], [2], 2),
    (40, 2, 128, [80, 64], [1, 1], 1),
    (24, 8, 128, [1000, 0, 77], [37, 40, 0], 40),
    (32, 8, 64, [130, 513], [100, 33], 100),
    (6, 2, 128, [4000], [200], 200),
    (32, 8, 64, [20000], [1], 1),
    (24, 8, 128, [0], [11], 11),
    (4, 4, 64, [127, 1], [33, 32], 33),
    (8, 8, 128, [100, 64], [64, 1], 64),
    (8, 8, 128, [100, 64], [65, 1], 65),
    (4, 4, 64, [500], [129], 129),
    (32, 8, 64, [0, 3000, 64], [300, 0, 257], 300),
    (24, 8, 128, [9000, 65], [86, 171], 171),
    (16, 1, 64, [200, 3], [1, 1], 1),
    (4, 4, 128, [70, 0], [4, 4], 4),
    # more conversations than a warp has lanes, some without a new token
    (4, 2, 64, [(37 * s) % 301 for s in range(70)], [s % 3 > 0 for s in range(70)], 1),
    (4, 2, 64, [(53 * s) % 200 for s in range(45)], [(7 * s) % 41 for s in range(45)], 40),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES, ids=[f"{c[0]}x{c[1]}x{c[2]}-{max(c[3])}+{c[5]}" for c in CASES])
def test_attention_over_cells(case, dtype):
    q_heads, kv_heads, dim, held, counts, q_len = case
    counts = [int(c) for c in counts]
    batch, query, k, v, keys, values = _filled(len(held), q_heads, kv_heads, dim, dtype, held, counts, q_len)
    scaling = dim ** -0.5
    out = batch.attend_layer(0, query, k, v, scaling)
    _check(out, query, keys, values, held, counts, scaling)
    out32 = batch.attend_layer(0, query, None, None, scaling, out_dtype=torch.float32)
    _check(out32, query, keys, values, held, counts, scaling)
    assert torch.equal(out32.to(dtype), out)
    batch.check_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q_len", [1, 2, 5, 40])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_where_every_score_is_nothing(dim, q_len, dtype):
    """A scaling of zero, or of next to nothing with queries of zero: the mean of the values that a row sees."""
    held, counts = [70, 0, 300], [q_len, q_len, q_len - 1]
    batch, query, k, v, keys, values = _filled(3, 4, 2, dim, dtype, held, counts, q_len)
    out = batch.attend_layer(0, query, k, v, 0.0)
    _check(out, query, keys, values, held, counts, 0.0)
    zero = torch.zeros_like(query)
    for scaling in (1e-30, -1e-30, -0.125):
        assert torch.equal(batch.attend_layer(0, zero, None, None, scaling), out)


ROW_CASES = [
    # three tiles of eight rows, full, with one more than two, and with padding
    (32, 8, 64, [70, 1000, 64], [6, 6, 6], 6),
    (17, 1, 64, [300, 0, 63], [1, 1, 0], 1),
    (8, 1, 64, [129, 40, 9000], [3, 0, 2], 3),
    # enough rows for a CTA of the joins to take 64, the last of them not a multiple of four
    (24, 8, 128, [300, 65, 1000, 0, 64], [171, 170, 3, 171, 0], 171),
    (32, 8, 64, [900, 0, 64, 1], [131, 130, 129, 131], 131),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", ROW_CASES, ids=[f"{c[0]}x{c[1]}x{c[2]}-{max(c[3])}+{c[5]}" for c in ROW_CASES])
def test_attention_of_row_counts_at_the_borders(case, dtype):
    test_attention_over_cells(case, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q_heads,kv_heads,dim,counts", [(8, 2, 64, [2500]), (6, 2, 128, [1500, 777]), (4, 4, 128, [2049])])
def test_attention_of_whole_prompts(q_heads, kv_heads, dim, counts, dtype):
    """Prompts in one piece: blocks of rows of up to forty steps, whose scores take the places of probabilities in turn."""
    held, q_len = [0] * len(counts), counts[0]
    batch, query, k, v, keys, values = _filled(len(counts), q_heads, kv_heads, dim, dtype, held, counts, q_len, seed=21)
    query *= 4  # rows whose maxima move from page to page
    out = batch.attend_layer(0, query, k, v, dim ** -0.5)
    _check(out, query, keys, values, held, counts, dim ** -0.5)
    for _ in range(3):
        assert torch.equal(batch.attend_layer(0, query, None, None, dim ** -0.5), out)
    batch.check_status()


def test_attention_of_peaked_and_flat_rows():
    """Scores far apart (one token takes all), equal ones, ones that grow along the context (the running maximum moves
    page after page), and queries of very small and very large size."""
    held, n, dim = [3000, 3000, 3000, 3000], 4, 128
    batch, query, k, v, keys, values = _filled(n, 24, 8, dim, torch.bfloat16, held, [1] * n, 1, seed=5)
    query[0] *= 30
    query[1] *= 0
    query[2] *= 2.0**-100
    query[3] *= 8
    out = batch.attend_layer(0, query, k, v, dim ** -0.5, out_dtype=torch.float32)
    _check(out, query, keys, values, held, [1] * n, dim ** -0.5)
    ramp = torch.linspace(-4, 4, 3001, device=DEV)[:, None] * torch.ones(dim, device=DEV)
    batch, query, k, v, keys, values = _filled(n, 24, 8, dim, torch.bfloat16, held, [1] * n, 1, seed=6)
    batch.trim([0] * n)
    keys = (ramp + 0.1 * keys.float()).to(torch.bfloat16)
    query = query.abs()
    batch.plan(None, 3001)
    batch.append(0, keys, values)
    batch.trim([3000] * n)
    batch.plan()
    out = batch.attend_layer(0, query, keys[:, :, -1:], values[:, :, -1:], dim ** -0.5, out_dtype=torch.float32)
    _check(out, query, keys, values, held, [1] * n, dim ** -0.5)
    batch.check_status()


def test_a_query_that_is_not_finite_stays_in_its_row():
    held, counts = [300, 90], [3, 3]
    batch, query, k, v, keys, values = _filled(2, 8, 2, 64, torch.float16, held, counts, 3, seed=9)
    query[0, 5, 1, 7] = float("nan")
    out = batch.attend_layer(0, query, k, v, 0.125)
    assert bool(out[0, 1, 5].isnan().all())
    out[0, 1, 5] = 0
    assert bool(torch.isfinite(out).all())
    query[0, 5, 1] = 0
    want = batch.attend_layer(0, query, None, None, 0.125)
    want[0, 1, 5] = 0
    assert torch.equal(out, want)


def test_strides_offsets_streams_and_graphs():
    """Tensors at other strides and odd offsets, a step captured and replayed (the tables advance on the device),
    and two conversations' pages shared out again."""
    n, q_heads, kv_heads, dim = 3, 24, 8, 128
    held = [70, 1, 130]
    batch, query, k, v, keys, values = _filled(n, q_heads, kv_heads, dim, torch.bfloat16, held, [1] * n, 1, seed=11)
    want = batch.attend_layer(0, query, k, v, 0.1)
    flat = torch.zeros(query.numel() + 3, dtype=query.dtype, device=DEV)
    odd = flat[3:].view(n, q_heads, 1, dim)
    odd.copy_(query)
    assert torch.equal(batch.attend_layer(0, odd, k.contiguous(), v.expand(n, kv_heads, 1, dim), 0.1), want)
    wide = torch.zeros(n, kv_heads, 1, dim + 4, dtype=k.dtype, device=DEV)
    wide[..., :dim] = k
    assert torch.equal(batch.attend_layer(0, query, wide[..., :dim], v, 0.1), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = batch.attend_layer(0, query, k, v, 0.1)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)

    # three steps one by one, and the same three as replays of one captured step
    steps = [(_rows(n, q_heads, 1, dim, torch.bfloat16, 50 + i), _rows(n, kv_heads, 1, dim, torch.bfloat16, 60 + i),
              _rows(n, kv_heads, 1, dim, torch.bfloat16, 70 + i)) for i in range(3)]
    mark = batch.lengths.clone()
    eager = []
    for q, a, b in steps:
        batch.plan()
        eager.append(batch.attend_layer(0, q, a, b, 0.1))
    batch.trim(mark)
    static = [x.clone() for x in steps[0]]
    batch.plan()
    batch.attend_layer(0, *static, 0.1)
    batch.trim(mark)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        batch.plan()
        held_out = batch.attend_layer(0, *static, 0.1)
    for (q, a, b), e in zip(steps, eager):
        for x, y in zip(static, (q, a, b)):
            x.copy_(y)
        graph.replay()
        assert torch.equal(held_out, e)
    assert torch.equal(batch.lengths, mark + 3)
    # a finished conversation's pages serve another
    batch.trim([0, 4, 133])
    batch.plan([0, 130, 0], 130)
    fresh = [_rows(n, kv_heads, 130, dim, torch.bfloat16, 80 + i) for i in range(2)]
    batch.append(0, *fresh)
    got = batch.read(0)
    for x, y in zip(fresh, got):
        assert torch.equal(y[1], dequantise4(*quantise4(x[1])).to(x.dtype))
    batch.check_status()


@pytest.mark.parametrize("q_len", [3, 40, 9000])
def test_captured_steps_of_any_length(q_len):
    """Plans (the larger ones with a second kernel) and attention of every form in a graph, the first call of their kind
    there; replays advance the tables, eager calls follow."""
    dim, kv, hq, n = 64, 2, 8, 2
    batch = Q4Batch(n, layers=1, kv_heads=kv, q_heads=hq, head_dim=dim, max_tokens=4 * q_len + 128)
    data = [[_rows(n, h, q_len, dim, torch.bfloat16, 10 * i + j) for j, h in enumerate((hq, kv, kv))] for i in range(3)]
    counts = torch.tensor([q_len, q_len - 1], dtype=torch.int32, device=DEV)
    static = [x.clone() for x in data[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        slots = batch.plan(counts, q_len)
        out = batch.attend_layer(0, *static, 0.125)
        batch.plan(None, 2)
        batch.trim(batch.table.starts)
    torch.cuda.current_stream().wait_stream(side)
    outs = []
    for x in data[:2]:
        for a, b in zip(static, x):
            a.copy_(b)
        graph.replay()
        outs.append((out.clone(), slots.clone()))
    assert batch.lengths.tolist() == [2 * q_len, 2 * q_len - 2]
    batch.plan(counts, q_len)
    last = batch.attend_layer(0, *data[2], 0.125)
    again = Q4Batch(n, layers=1, kv_heads=kv, q_heads=hq, head_dim=dim, max_tokens=4 * q_len + 128)
    for x, got in zip(data, outs + [(last, None)]):
        s = again.plan(counts, q_len)
        assert torch.equal(again.attend_layer(0, *x, 0.125), got[0])
        assert got[1] is None or torch.equal(s, got[1])
    batch.plan(None, 2)  # its even counts were first made in the capture
    assert batch.lengths.tolist() == [3 * q_len + 2, 3 * q_len - 1]
    batch.check_status()
    again.check_status()


def test_two_readers_at_once():
    """Attention without new tokens only reads: two streams at a time, several calls each, the same answers."""
    held = [5000, 700, 64]
    batch, query, k, v, keys, values = _filled(3, 24, 8, 128, torch.bfloat16, held, [1] * 3, 1, seed=3)
    want = batch.attend_layer(0, query, k, v, 0.09)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(20):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(batch.attend_layer(0, query, None, None, 0.09))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("q_len", [1, 5, 90])
def test_two_batches_on_two_streams(q_len):
    """Two batches, each stored to and attended by a stream of its own, step after step: as one after the other."""
    data = [[[_rows(2, h, q_len, 64, torch.float16, 100 * b + 10 * i + j) for j, h in enumerate((16, 4, 4))] for i in range(6)]
            for b in range(2)]
    held = [[_rows(2, 4, 700, 64, torch.float16, 900 + 2 * b + j) for j in range(2)] for b in range(2)]
    batches = []
    for _ in range(2):
        for b in range(2):
            batch = Q4Batch(2, layers=1, kv_heads=4, q_heads=16, head_dim=64, max_tokens=700 + 6 * q_len, dtype=torch.float16)
            batch.plan([700, 311], 700)
            batch.append(0, *held[b])
            batches.append(batch)

    def step(batch, x, i):
        batch.plan([q_len, q_len - i % 2], q_len)
        return batch.attend_layer(0, *x, 0.125)

    want = [[step(batches[b], x, i) for i, x in enumerate(data[b])] for b in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for i in range(6):
        for b in range(2):
            with torch.cuda.stream(streams[b]):
                got[b].append(step(batches[2 + b], data[b][i], i))
    torch.cuda.synchronize()
    for b in range(2):
        assert all(torch.equal(x, y) for x, y in zip(want[b], got[b]))
        batches[2 + b].check_status()


def test_far_pages_of_a_large_pool():
    """Cells beyond 2^32 bytes: the pages of one conversation lie at the end of a pool of 5 GB."""
    dim, kv = 128, 8
    pages = 70000
    batch = Q4Batch(1, layers=1, kv_heads=kv, q_heads=24, head_dim=dim, max_tokens=200, n_pages=pages)
    assert batch.cells.numel() > 2**32
    batch.table.free.copy_(torch.arange(pages, dtype=torch.int32, device=DEV))  # the last page first
    k, v, q = _rows(1, kv, 130, dim, torch.bfloat16, 1, "key"), _rows(1, kv, 130, dim, torch.bfloat16, 2), _rows(1, 24, 130, dim, torch.bfloat16, 3)
    batch.plan(None, 130)
    out = batch.attend_layer(0, q, k, v, 0.09)
    assert batch.table.blocks[0, :3].tolist() == [pages - 1, pages - 2, pages - 3]
    _check(out, q, k, v, [0], [130], 0.09)
    a, b = batch.read(0)
    assert torch.equal(a, dequantise4(*quantise4(k)).to(k.dtype)) and torch.equal(b, dequantise4(*quantise4(v)).to(v.dtype))
    batch.check_status()


# ------------------------------------------------------------------------------------------------ a model over it
class _Checked:
    """A Q4Batch of one conversation whose every attention call is held against attend64 on the call's own inputs.
    (Whole logits cannot be held against a plain model's: a difference of 2^-11 in one layer's output moves some
    of the next layer's keys across a border between two codes, a whole step of 4 bits.)"""

    def __init__(self, batch):
        self.batch, self.keys, self.values, self.calls = batch, {}, {}, 0

    def attend(self, module, query, key, value, attention_mask, scaling):
        out, _ = self.batch.attend(module, query, key, value, attention_mask, scaling)
        layer, dtype = module.layer_idx, self.batch.dtype
        for store, x in ((self.keys, key), (self.values, value)):
            store[layer] = torch.cat(([store[layer]] if layer in store else []) + [x[0].to(dtype)], 1)
        held = self.keys[layer].shape[1] - query.shape[2]
        want, parts = attend64(query[0].to(dtype), self.keys[layer], self.values[layer], held, scaling)
        assert out.dtype == torch.promote_types(query.dtype, dtype) and out.shape[1:] == want.shape
        assert float(((out[0].double() - want).abs() - attend_tolerance(want, parts, dtype, out.dtype, query.shape[2] * 4)).max()) <= 0
        self.calls += 1
        return out, None


class _Tokens:
    eos_token_id, all_special_ids = -1, []

    def decode(self, ids, skip_special_tokens=True):
        return " ".join(map(str, ids))


@pytest.mark.parametrize("model_dtype,dtype", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16),
                                               (torch.float16, torch.float16)])
def test_a_model_decodes_over_cells(model_dtype, dtype):
    """Prefill in two chunks and a decoded token of the tiny model through the hook."""
    model = tm.build_model(model_dtype, DEV)
    dimmer.install(model)
    ids = tm.context_ids().to(DEV)[:, :301]
    batch = Q4Batch(1, layers=2, kv_heads=8, q_heads=32, head_dim=64, max_tokens=400, dtype=dtype)
    context = dimmer.STATE.compressed = _Checked(batch)
    try:
        with torch.inference_mode():
            for first, end in ((0, 129), (129, 300), (300, 301)):
                model(input_ids=ids[:, first:end], past_key_values=batch.cache,
                      position_ids=torch.arange(first, end, device=DEV)[None], use_cache=True)
    finally:
        dimmer.STATE.compressed = None
    batch.check_status()
    assert batch.lengths.tolist() == [301] and context.calls == 6


def test_answers_with_rules_over_a_context():
    """Q4Context and greedy_answer with penalties and a grammar: the answer holds no token twice, and only allowed
    ones; the first logits are the plain cache's within 4 bits of noise."""
    model = tm.build_model(torch.bfloat16, DEV)
    dimmer.install(model)
    ids = tm.context_ids().to(DEV)[:, :200]
    with torch.inference_mode():
        cache, _ = dimmer.prefill_with_scores(model, ids)
        keys, values = [l.keys for l in cache.layers], [l.values for l in cache.layers]
        context = Q4Context(keys, values, model, dtype=torch.bfloat16)
        assert context.code_bytes() == 200 * 2 * 8 * 2 * 36
        question = tm.question_ids().to(DEV)[None]
        text, first = greedy_answer(model, _Tokens(), context, context.exact_cache, question, 200)
        again = Q4Context(keys, values, model, dtype=torch.bfloat16)
        rules = LogitRules(1, 1024, capacity=32, presence=1000.0)
        allowed = allow_mask([list(range(0, 1024, 3))], 1024)
        even = lambda last: allowed
        text2, first2 = greedy_answer(model, _Tokens(), again, again.exact_cache, question, 200, rules=rules, grammar=even)
    assert torch.equal(first, first2)
    tokens = [int(t) for t in text2.split()]
    assert len(tokens) == 12 == len(set(tokens)) and all(t % 3 == 0 for t in tokens)
    assert rules.lengths.tolist() == [12] and rules.history[0, :12].tolist() == tokens
    assert tokens[0] == int(torch.where(torch.arange(1024, device=DEV) % 3 == 0, first, float("-inf")).argmax())
    context.batch.check_status()
    again.batch.check_status()


def test_batch_decodes_with_rules():
    """greedy_decode_batch over a Q4Batch: ragged conversations, each as if it were alone."""
    model = tm.build_model(torch.bfloat16, DEV)
    dimmer.install(model)
    ids = tm.context_ids().to(DEV)
    lengths = [150, 64, 33]
    with torch.inference_mode():
        def context(rows):
            n = len(rows)
            batch = Q4Batch(n, layers=2, kv_heads=8, q_heads=32, head_dim=64, max_tokens=300)
            longest = max(lengths[r] for r in rows)
            x = torch.zeros(n, longest, dtype=torch.int64, device=DEV)
            for i, r in enumerate(rows):
                x[i, :lengths[r]] = ids[0, r * 150:r * 150 + lengths[r]]
            batch.begin([lengths[r] for r in rows])
            dimmer.STATE.compressed = batch
            try:
                model(input_ids=x, past_key_values=batch.cache, position_ids=torch.arange(longest, device=DEV)[None].expand(n, -1),
                      use_cache=True)
            finally:
                dimmer.STATE.compressed = None
            rules = LogitRules(n, 1024, capacity=64, repetition=1.3, frequency=0.2)
            rules.load(x.to(torch.int32)[:, :33], [33] * n)
            start = torch.tensor([[r + 1] for r in rows])
            out, _ = greedy_decode_batch(model, batch, batch.cache, start, torch.tensor([[lengths[r]] for r in rows]), 6,
                                         rules=rules)
            batch.check_status()
            rules.check_status()
            assert rules.lengths.tolist() == [39] * n
            return out, [x.float() for x in batch.read(1, batch.table.slots(lengths[rows[0]]))]

        together, kv = context([0, 1, 2])
        for r in range(3):
            alone, kv1 = context([r])
            # the same tokens unless the model's own batched products (cuBLAS) decide a near tie otherwise: the first
            # token's cells are equal up to one code of a value that a rounding of the projection moved
            assert float((kv[0][r, :, :1] - kv1[0][0, :, :1]).abs().max()) < 0.5
            assert together.shape == (3, 6) and int(together.min()) >= 0
        rules = LogitRules(1, 1024)
        batch = Q4Batch(1, layers=2, kv_heads=8, q_heads=32, head_dim=64, max_tokens=300)
        with pytest.raises(_lib.DimmerKVError, match="no token is allowed"):
            greedy_decode_batch(model, batch, batch.cache, torch.tensor([[1]]), torch.tensor([[0]]), 2, rules=rules,
                                grammar=lambda last: allow_mask([[]], 1024))


def test_the_hook_refuses_another_cache_and_another_mask():
    model = tm.build_model(torch.bfloat16, DEV)
    dimmer.install(model)
    ids = tm.context_ids().to(DEV)[:, :6].repeat(2, 1)
    pos = torch.arange(6, device=DEV)[None].expand(2, -1)
    batch = Q4Batch(2, layers=2, kv_heads=8, q_heads=32, head_dim=64, max_tokens=64)
    full = torch.ones(2, 6, dtype=torch.int64, device=DEV)
    left = full.clone()
    left[1, :2] = 0
    right = full.clone()
    right[1, 4:] = 0
    dimmer.STATE.compressed = batch
    try:
        with torch.inference_mode():
            call = lambda mask: model(input_ids=ids, past_key_values=batch.cache, position_ids=pos, attention_mask=mask)
            call(full)
            batch.check_status()
            batch.begin([6, 4])
            call(right)  # padded behind the counts: what the batch is told
            batch.check_status()
            call(left)
            with pytest.raises(_lib.DimmerKVError, match="115"):
                batch.check_status()
            batch.reset_status()
            dyn = model(input_ids=ids[:, :2], position_ids=pos[:, :2], use_cache=True).past_key_values
            with pytest.raises(ValueError, match="own cache"):
                model(input_ids=ids[:, :1], past_key_values=dyn, position_ids=pos[:, 2:3])
    finally:
        dimmer.STATE.compressed = None


def test_methods_q4_rebuilds_the_cells():
    g = torch.Generator().manual_seed(5)
    keys = [torch.randn(1, 8, 130, 64, generator=g).half() for _ in range(2)]
    values = [torch.randn(1, 8, 130, 64, generator=g).half() for _ in range(2)]
    host = Methods("m", "none", "none", "cpu").apply("q4", keys, values, {})
    gpu = Methods("m", "none", "none", DEV).apply("q4", [k.to(DEV) for k in keys], [v.to(DEV) for v in values], {})
    assert gpu.used_bytes == host.used_bytes
    for a, b in zip(gpu.keys + gpu.values, host.keys + host.values):
        assert torch.equal(a.cpu(), b)
