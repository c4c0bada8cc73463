"""The paged 4-bit cache and the logit rules without a GPU: the quantiser in torch operations, the refusals, the
masks, and what the methods rebuild."""

from __future__ import annotations

import ctypes

import pytest
import torch

from dimmerkv import _lib, q4
from dimmerkv.compressed_attention import greedy_answer, greedy_decode_batch
from dimmerkv.logits import LogitRules, allow_mask
from dimmerkv.methods import Methods
from dimmerkv.paging import PageTable
from dimmerkv.q4 import Q4Batch, dequantise4, quantise4
from q4_reference import PlainTable, cells64

needs_lib = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="library not built (dimmer-kv_b200/build_lib.py)")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantise4_is_the_definition(dtype):
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(5, 3, 128, generator=g) * torch.logspace(-3, 2, 128)).to(dtype)
    x[0, 0] = 0.25           # a constant group: every code 0, value = low
    x[1, 0, :64] = -7.0
    codes, scale, low = quantise4(x)
    want, s64, l64 = cells64(x)
    assert torch.equal(scale.double(), s64) and torch.equal(low.double(), l64)
    got = dequantise4(codes, scale, low).double()
    # one float32 rounding of the sum against the exact one
    assert bool(((got - want).abs() <= want.abs() * 2**-24).all())
    # 4 bits hold x to half a step (and low's own rounding, which the codes see)
    step = s64.repeat_interleave(64, -1)
    cut = (l64.abs() * 2**-11).repeat_interleave(64, -1)
    top = (x.double() - want).abs() - step / 2 - cut - step * 15 * 2**-11
    assert float(top.max()) <= 1e-7  # float16's subnormal step


def test_methods_q4_on_the_host():
    g = torch.Generator().manual_seed(5)
    keys = [torch.randn(1, 2, 9, 64, generator=g).half() for _ in range(3)]
    values = [torch.randn(1, 2, 9, 64, generator=g).half() for _ in range(3)]
    out = Methods("m", "none", "none", "cpu").apply("q4", keys, values, {})
    for a, b in zip(out.keys + out.values, keys + values):
        assert torch.equal(a, cells64(b)[0].float().half())
    assert out.used_bytes == 3 * 2 * 2 * 9 * (32 + 4)
    assert out.token_bytes.shape == (9,) and float(out.token_bytes.sum()) == out.used_bytes


def test_table_refusals():
    for bad in (dict(n_seq=0), dict(n_seq=8193), dict(n_pages=0), dict(max_tokens=0), dict(max_tokens=2**31),
                dict(n_pages=2**25 + 1), dict(free=torch.zeros(3)), dict(free=torch.zeros(9, dtype=torch.int32)),
                dict(device="cpu")):
        with pytest.raises(ValueError):
            PageTable(**{**dict(n_seq=2, n_pages=8, max_tokens=100), **bad})


def test_batch_refusals():
    base = dict(layers=1, kv_heads=2, q_heads=4, head_dim=64, max_tokens=64)
    with pytest.raises(NotImplementedError):
        Q4Batch(1, **{**base, "head_dim": 96})
    for bad in (dict(q_heads=3), dict(layers=0), dict(kv_heads=0), dict(dtype=torch.float32), dict(device="cpu")):
        with pytest.raises(ValueError):
            Q4Batch(1, **{**base, **bad})


def test_rules_refusals():
    ids, vals = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 3)
    for bad in (dict(n_rows=0), dict(vocab=0), dict(capacity=0), dict(repetition=0.0), dict(repetition=float("nan")),
                dict(bias_ids=ids), dict(bias_ids=ids, bias_values=vals[:, :2]),
                dict(bias_ids=ids[:1], bias_values=vals[:1]),
                dict(bias_ids=torch.zeros(2, 1025, dtype=torch.int32), bias_values=torch.zeros(2, 1025)),
                dict(presence=torch.zeros(3)), dict(device="cpu")):
        with pytest.raises(ValueError):
            LogitRules(**{**dict(n_rows=2, vocab=10), **bad})
    with pytest.raises(ValueError):
        allow_mask([[10]], 10, "cpu")
    with pytest.raises(ValueError):
        greedy_answer(None, None, None, None, torch.zeros(1, 1), 0, grammar=lambda last: None)
    with pytest.raises(ValueError):
        greedy_decode_batch(None, None, None, None, None, 1, grammar=lambda last: None)


def test_allow_mask_bits():
    m = allow_mask([[0, 31, 32, 66], []], 67, "cpu")
    assert m.shape == (2, 3) and m.dtype == torch.int32
    assert [int(v) & 0xffffffff for v in m[0]] == [0x80000001, 1, 4] and not m[1].any()


@needs_lib
def test_entry_points_refuse_on_the_host():
    """Arguments that a kernel must never see come back as codes before any CUDA call."""
    lib = _lib.lib()
    assert [lib.dkv_q4_page_bytes(d) for d in (64, 128, 96)] == [4608, 9216, -1]
    p = 1 << 20  # never followed
    table = dict(blocks=p, max_blocks=2, lengths=p, starts=p, free_pages=p, n_free=p, n_pages=4, n_seq=1, counts=p,
                 q_len=1, slots=p, status=p)
    for name, bad, rc in (("plan", dict(blocks=None), 1), ("plan", dict(slots=None), 1), ("plan", dict(q_len=-1), 1),
                          ("plan", dict(n_seq=8193), 2), ("plan", dict(n_pages=1 << 26), 2), ("plan", dict(n_pages=0), 1),
                          ("trim", dict(free_pages=None), 1), ("trim", dict(max_blocks=0), 1),
                          ("slots", dict(counts=None), 1), ("plan", dict(n_seq=0), 0), ("slots", dict(q_len=0), 0)):
        a = _lib.PageArgs(**{**table, **bad})
        assert getattr(lib, f"dkv_page_{name}")(a, None) == rc, (name, bad)
    i64 = ctypes.c_int64 * 3
    rows = dict(cells=p, n_pages=4, n_kv_heads=2, head_dim=64, fp16=0, slots=p, n_seq=1, q_len=1, key=p, value=p,
                k_stride=i64(8, 8, 8), v_stride=i64(8, 8, 8), status=p)
    for bad, rc in ((dict(cells=p + 1), 1), (dict(key=p + 2), 1), (dict(k_stride=i64(8, 4, 8)), 1),
                    (dict(head_dim=80), 2), (dict(value=None), 1), (dict(n_pages=1 << 26), 2), (dict(q_len=0), 0)):
        for fn in (lib.dkv_q4_append, lib.dkv_q4_read):
            assert fn(_lib.Q4RowsArgs(**{**rows, **bad}), None) == rc, bad
    att = dict(cells=p, n_pages=4, n_kv_heads=2, n_q_heads=4, head_dim=64, fp16=0, blocks=p, max_blocks=1, lengths=p,
               starts=p, n_seq=1, q_len=1, len_bound=64, query=p, q_stride=i64(8, 8, 8), scaling=1.0, out=p, out_f32=0,
               workspace=p, workspace_floats=1 << 40, status=p)
    for bad, rc in ((dict(n_q_heads=3), 1), (dict(key=p), 1), (dict(key=p, value=p), 1), (dict(workspace=None), 5),
                    (dict(workspace_floats=100), 5), (dict(out=p + 4), 1), (dict(n_seq=8193), 2),
                    (dict(key=p, value=p, slots=p, v_stride=i64(8, 8, 1)), 1), (dict(query=p + 8), 1), (dict(q_stride=i64(8, 8, 12)), 1),
                    (dict(head_dim=32), 2), (dict(status=None), 1), (dict(q_len=-1), 1), (dict(n_seq=70000), 2),
                    (dict(n_seq=0), 0), (dict(q_len=0), 0)):
        assert lib.dkv_q4_attend(_lib.Q4AttendArgs(**{**att, **bad}), None) == rc, bad
    log = dict(logits=p, dtype=0, row_stride=10, n_rows=1, vocab=10, history=p, capacity=4, lengths=p, prompts=p,
               repetition=p, frequency=p, presence=p, tokens=p, status=p)
    for bad, rc in ((dict(dtype=3), 1), (dict(vocab=0), 1), (dict(n_bias=2), 1), (dict(tokens=None), 1),
                    (dict(n_bias=1025, bias_ids=p, bias_values=p), 2), (dict(row_stride=-1), 1), (dict(n_rows=0), 0)):
        assert lib.dkv_logit_rules(_lib.LogitsArgs(**{**log, **bad}), None) == rc, bad


def test_plain_table_undoes_a_plan():
    """The rule that the kernels follow: trim(starts) gives the pages back in the order that plan took them."""
    t = PlainTable(3, 20, 400)
    t.plan([70, 3, 200], 200)
    free, blocks = list(t.free), t.array().copy()
    t.plan([100, 0, 64], 100)
    t.trim(list(t.starts))
    assert t.free == free and (t.array() == blocks).all()


def test_struct_mirrors_of_the_new_entry_points():
    import re

    from test_abi_cpu import HEADER

    text = HEADER.read_text()
    for struct, mirror in (("dkv_page_args", _lib.PageArgs), ("dkv_q4_rows_args", _lib.Q4RowsArgs),
                           ("dkv_q4_attend_args", _lib.Q4AttendArgs), ("dkv_logits_args", _lib.LogitsArgs)):
        body = re.search(r"typedef struct " + struct + r" \{(.*?)\} " + struct + ";", text, flags=re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        names = [re.sub(r"\[.*?\]", "", f).split()[-1].lstrip("*") for stmt in body.split(";") if stmt.strip()
                 for f in stmt.split(",")]
        assert names == [f[0] for f in mirror._fields_], struct


def test_scales_have_no_sign():
    """Groups whose least value, rounded to float16, lies above their largest: code 0 of a scale of +0."""
    x = torch.full((3, 64), -1e-8).bfloat16()
    x[1] = -1.5e-6
    x[2, ::2] = -1.4e-6
    codes, scale, low = quantise4(x)
    assert bool((low.float()[:, 0] >= x.float().amax(-1)).any())
    assert not scale.signbit().any() and not codes[:2].any()
    assert torch.equal(dequantise4(codes, scale, low).double(), cells64(x)[0])


@needs_lib
def test_entry_points_take_calls_without_a_token():
    """Tensors without an element have no address: such calls do nothing, and their sizes are checked all the same."""
    lib = _lib.lib()
    p = 1 << 20  # never followed
    rows = dict(cells=p, n_pages=4, n_kv_heads=2, head_dim=64, n_seq=1, q_len=0, status=p)
    att = dict(cells=p, n_pages=4, n_kv_heads=2, n_q_heads=4, head_dim=64, blocks=p, max_blocks=1, lengths=p, starts=p, n_seq=1,
               q_len=0, len_bound=64, scaling=1.0, status=p)
    table = dict(blocks=p, max_blocks=2, lengths=p, starts=p, n_seq=1, counts=p, q_len=0, status=p)
    for bad, rc in ((dict(), 0), (dict(n_seq=0, q_len=3), 0), (dict(head_dim=96), 2), (dict(n_kv_heads=0), 1),
                    (dict(q_len=1), 1), (dict(cells=None), 1)):
        for fn in (lib.dkv_q4_append, lib.dkv_q4_read):
            assert fn(_lib.Q4RowsArgs(**{**rows, **bad}), None) == rc, bad
        a = _lib.Q4AttendArgs(**{**att, **bad})
        assert lib.dkv_q4_attend(a, None) == rc, bad
    assert lib.dkv_q4_attend_floats(_lib.Q4AttendArgs(**att)) == 0
    assert lib.dkv_page_slots(_lib.PageArgs(**table), None) == 0


def test_tables_refuse_free_lists_that_share_pages():
    """A page that is listed twice would serve two conversations, one that the pool does not have none."""
    for free in ([3, 3], [0, 8], [-1, 2], list(range(7)) + [0]):
        with pytest.raises(ValueError, match="free"):
            PageTable(2, 8, 100, free=torch.tensor(free, dtype=torch.int32), device="cpu")
    for free in ([], [7, 0], list(range(8))):
        with pytest.raises(ValueError, match="CUDA device"):  # (only the device is wrong)
            PageTable(2, 8, 100, free=torch.tensor(free, dtype=torch.int32), device="cpu")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 40000.0, -32800.0])
def test_values_without_a_cell_are_refused_on_the_host(bad, dtype):
    """As on the GPU: a group that 4 bits cannot hold is no cache of zeros, infinities or NaN."""
    keys = [torch.ones(1, 2, 3, 64, dtype=dtype) for _ in range(2)]
    values = [k.clone() for k in keys]
    values[1][0, 1, 2, 63] = -32768.0 if dtype != torch.float32 else 32768.0  # the largest that a cell holds
    q4.restore(keys, values)
    values[1][0, 1, 2, 63] = bad
    if abs(float(values[1].amin())) == 32768.0:  # bfloat16 has steps of 256 there: -32800 is -32768 to it
        assert dtype == torch.bfloat16 and bad == -32800.0
        return
    with pytest.raises(_lib.DimmerKVError, match="4-bit cell"):
        q4.restore(keys, values)
    with pytest.raises(_lib.DimmerKVError, match="4-bit cell"):
        Methods("m", "none", "none", "cpu").apply("q4", values, keys, {})
    q4.restore([k[:, :, :0] for k in keys], [v[:, :, :0] for v in values])
