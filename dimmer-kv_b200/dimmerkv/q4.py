"""The paged 4-bit cache: keys and values of a batch of conversations in 4 bits, and attention over them.

Where ``CompressedBatch`` needs a fitted basis and codes made after the prefill, this cache takes tokens as they
come: every group of 64 dimensions of a token's key or value is kept as 4-bit codes with a float16 scale and low
(4.5 bits per element), in pages of 64 tokens that the conversations share (``paging.PageTable``).

``Q4Batch`` plugs into the attention hook like ``CompressedBatch`` (``dimmer.STATE.compressed``, ``greedy_answer``,
``greedy_decode_batch``): a forward pass stores its new tokens and attends over all of them. Its ``cache`` stands in
for the Hugging Face cache of such a pass: it hands the new keys and values on and keeps none. ``Q4Context`` is
the one-conversation form with the constructor of ``CompressedContext``.

The cache serves: no gradients flow through it. Calls that change a batch (``plan``, ``append``, ``attend``) follow
one another in stream order, on one stream or on streams that the caller joins.
"""

from __future__ import annotations

import torch
from transformers import DynamicCache

from . import _lib
from .paging import PAGE, PageTable, pages_of

GROUP = 64
CELL_MAX = 32768.0  # largest magnitude that a cell holds
CELL_ERROR, MASK_ERROR = 8113, 115


def cell_bytes(head_dim: int) -> int:
    """Bytes of one token's keys (or values) of one KV head: 4-bit codes, float16 scale and low per 64."""
    return head_dim // 2 + head_dim // GROUP * 4


def quantise4(x: torch.Tensor):
    """[..., dim] -> codes uint8 [..., dim] (0..15), scale and low float16 [..., dim / 64]: what ``append`` stores,
    in torch operations, on any device."""
    g = x.float().unflatten(-1, (-1, GROUP))
    low = g.amin(-1).half()
    scale = ((g.amax(-1) - low.float()).clamp_min(0.0) / 15).half().abs()  # low may round above the largest: +0
    step = scale.double()[..., None]
    q = (g.double() - low.double()[..., None]) / torch.where(step > 0, step, torch.ones_like(step))
    q = torch.where(step > 0, q.round().clamp(0, 15), torch.zeros_like(q))
    return q.to(torch.uint8).flatten(-2), scale, low


def dequantise4(codes: torch.Tensor, scale: torch.Tensor, low: torch.Tensor) -> torch.Tensor:
    """The float32 values of ``quantise4``'s codes."""
    g = codes.float().unflatten(-1, (-1, GROUP))
    return (g * scale.float()[..., None] + low.float()[..., None]).flatten(-2)


class Q4Cache(DynamicCache):
    """The Hugging Face cache of a forward pass over a ``Q4Batch``: new keys and values pass through to the
    attention hook, which stores them in 4 bits. Positions are the caller's (``position_ids``), as in
    ``greedy_answer``."""

    def update(self, key_states, value_states, layer_idx, *args, **kwargs):
        return key_states, value_states


class Q4Batch:
    """4-bit keys and values of ``n_seq`` conversations of up to ``max_tokens`` tokens.

    ``n_pages`` pages of 64 tokens are shared by the conversations (default: enough for all of them at full
    length). ``dtype`` is the 16-bit type of queries, keys, values and outputs (bfloat16 or float16)."""

    def __init__(self, n_seq: int, *, layers: int, kv_heads: int, q_heads: int, head_dim: int, max_tokens: int,
                 n_pages: int | None = None, device="cuda", dtype=torch.bfloat16):
        if head_dim not in (64, 128):
            raise NotImplementedError(f"the 4-bit cache handles head_dim 64 and 128, not {head_dim}")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("dtype must be torch.bfloat16 or torch.float16")
        if layers < 1 or kv_heads < 1 or q_heads < 1 or q_heads % kv_heads:
            raise ValueError("layers and kv_heads must be at least 1, q_heads a multiple of kv_heads")
        self.table = PageTable(n_seq, n_seq * pages_of(max_tokens) if n_pages is None else n_pages, max_tokens, device)
        self.device, self.dtype = self.table.device, dtype
        self.n_seq, self.layers, self.kv_heads, self.q_heads, self.head_dim = n_seq, layers, kv_heads, q_heads, head_dim
        self.lib = _lib.lib()
        self.status = self.table.status
        self.cells = torch.zeros(layers, self.table.n_pages, kv_heads, int(self.lib.dkv_q4_page_bytes(head_dim)),
                                 dtype=torch.uint8, device=self.device)
        self.cache = Q4Cache()
        self._slots = None   # of the newest plan
        self._counts = None  # of the next forward pass (begin)
        self._rows = _lib.Q4RowsArgs()
        r = self._rows
        r.n_pages, r.n_kv_heads, r.head_dim, r.fp16 = self.table.n_pages, kv_heads, head_dim, int(dtype == torch.float16)
        r.n_seq, r.status = n_seq, self.status.data_ptr()
        self._attend = _lib.Q4AttendArgs()
        a = self._attend
        a.n_pages, a.n_kv_heads, a.n_q_heads, a.head_dim = self.table.n_pages, kv_heads, q_heads, head_dim
        a.fp16, a.blocks, a.max_blocks = r.fp16, self.table.blocks.data_ptr(), self.table.max_blocks
        a.lengths, a.starts, a.n_seq = self.table.lengths.data_ptr(), self.table.starts.data_ptr(), n_seq
        a.status = self.status.data_ptr()
        self._calls: dict[tuple, _lib.Q4AttendArgs] = {}
        self._layer_bytes = self.cells[0].numel()
        self._cells_ptr = self.cells.data_ptr()

    # ------------------------------------------------------------------ tokens
    @property
    def lengths(self) -> torch.Tensor:
        return self.table.lengths

    def token_bytes(self) -> int:
        """Bytes that one token takes over all layers."""
        return self.layers * self.kv_heads * 2 * cell_bytes(self.head_dim)

    def plan(self, counts=None, q_len: int = 1) -> torch.Tensor:
        """Room for the next tokens of every conversation (``PageTable.plan``); ``append`` and ``attend_layer``
        then take them in rows of ``q_len``, conversation s its first ``counts[s]``."""
        self._slots = self.table.plan(counts, q_len)
        return self._slots

    def trim(self, keep) -> None:
        """Keep the first ``keep[s]`` tokens of every conversation (0: its pages are free for others)."""
        self.table.trim(keep)
        self._slots = None

    def _layer(self, layer: int) -> int:
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} of {self.layers}")
        return self._cells_ptr + layer * self._layer_bytes

    def _check(self, name: str, x: torch.Tensor, heads: int, rows: int) -> None:
        if x.shape != (self.n_seq, heads, rows, self.head_dim):
            raise ValueError(f"{name} {tuple(x.shape)} is not [{self.n_seq}, {heads}, {rows}, {self.head_dim}]")
        if x.device != self.device:
            raise ValueError(f"{name} is on {x.device}, the cache on {self.device}")

    def _tensor(self, name: str, x: torch.Tensor, heads: int, rows: int):
        """x [n_seq, heads, rows, head_dim] as the kernels take it, and its strides."""
        self._check(name, x, heads, rows)
        if x.dtype is not self.dtype:
            x = x.to(self.dtype)
        strides = x.stride()
        if strides[3] != 1 or (strides[0] | strides[1] | strides[2]) % 8 or x.data_ptr() % 16:
            # the stride of a dimension of one is free
            strides = tuple(s if n > 1 else 0 for s, n in zip(strides, x.shape[:3])) + (strides[3],)
            if strides[3] != 1 or (strides[0] | strides[1] | strides[2]) % 8 or x.data_ptr() % 16:
                x = x.contiguous()
                if x.data_ptr() % 16:
                    x = x.clone()
                strides = x.stride()
        return x, strides[:3]

    def append(self, layer: int, key: torch.Tensor, value: torch.Tensor) -> None:
        """Store key / value [n_seq, kv_heads, q_len, head_dim] of the planned tokens in one layer's cells."""
        if self._slots is None:
            raise RuntimeError("append needs the slots of a plan")
        cells = self._layer(layer)
        q_len = self._slots.shape[1]
        a = _lib.Q4RowsArgs.from_buffer_copy(self._rows)
        key, a.k_stride = self._tensor("key", key, self.kv_heads, q_len)
        value, a.v_stride = self._tensor("value", value, self.kv_heads, q_len)
        a.cells, a.slots, a.q_len = cells, self._slots.data_ptr(), q_len
        a.key, a.value = key.data_ptr(), value.data_ptr()
        _lib.launch("dkv_q4_append", a, self.device)

    def read(self, layer: int, slots: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The keys and values that the cells of ``slots`` (int32 [n_seq, n]; default: the newest plan's) stand
        for, [n_seq, kv_heads, n, head_dim], zeros for slot -1."""
        slots = self._slots if slots is None else slots
        if slots is None:
            raise RuntimeError("read needs slots, or a plan before it")
        if slots.dtype != torch.int32 or slots.device != self.device or slots.dim() != 2 or slots.shape[0] != self.n_seq:
            raise ValueError(f"slots must be int32 [{self.n_seq}, n] on {self.device}")
        slots = slots.contiguous()
        a = _lib.Q4RowsArgs.from_buffer_copy(self._rows)
        n = slots.shape[1]
        key, value = torch.empty(2, self.n_seq, self.kv_heads, n, self.head_dim, dtype=self.dtype,
                                 device=self.device).unbind(0)
        a.cells, a.slots, a.q_len = self._layer(layer), slots.data_ptr(), n
        a.key, a.value = key.data_ptr(), value.data_ptr()
        a.k_stride = a.v_stride = key.stride()[:3]
        _lib.launch("dkv_q4_read", a, self.device)
        return key, value

    # ------------------------------------------------------------------ attention
    def attend_layer(self, layer: int, query: torch.Tensor, key: torch.Tensor | None, value: torch.Tensor | None,
                     scaling: float, out_dtype=None) -> torch.Tensor:
        """Store the planned tokens' key / value [n_seq, kv_heads, q_len, head_dim] (``None``: they are stored) and
        attend with their queries [n_seq, q_heads, q_len, head_dim], causally, over every token of their
        conversation. Returns [n_seq, q_len, q_heads, head_dim] in the cache dtype (or float32 with
        ``out_dtype=torch.float32``), zeros behind a conversation's new tokens."""
        out_dtype = out_dtype or self.dtype
        if out_dtype not in (self.dtype, torch.float32):
            raise ValueError(f"out_dtype must be {self.dtype} or torch.float32")
        if (key is None) != (value is None):
            raise ValueError("key and value come together")
        if self._slots is None:
            raise RuntimeError("attend_layer needs a plan")
        q_len = self._slots.shape[1]
        query, q_stride = self._tensor("query", query, self.q_heads, q_len)
        strides = (q_len, out_dtype, q_stride)
        if key is not None:
            key, k_stride = self._tensor("key", key, self.kv_heads, q_len)
            value, v_stride = self._tensor("value", value, self.kv_heads, q_len)
            strides += (k_stride, v_stride)
        made = self._calls.get(strides)
        if made is None:  # what stays the same from call to call of this form
            made = _lib.Q4AttendArgs.from_buffer_copy(self._attend)
            made.q_len, made.q_stride, made.out_f32 = q_len, q_stride, int(out_dtype == torch.float32)
            if key is not None:
                made.k_stride, made.v_stride = k_stride, v_stride
            made.workspace_floats = int(self.lib.dkv_q4_attend_floats(made))
            if len(self._calls) > 64:
                self._calls.clear()
            self._calls[strides] = made
        a = _lib.Q4AttendArgs.from_buffer_copy(made)
        out = torch.empty((self.n_seq, q_len, self.q_heads, self.head_dim), dtype=out_dtype, device=self.device)
        workspace = torch.empty(a.workspace_floats, dtype=torch.float32, device=self.device)
        # a captured call serves whatever lengths the tables have when it is replayed: one that was split for the 64 tokens at
        # its capture took 49 us over 16384 tokens (24 / 8 heads of 128) where 16 are enough
        bound = self.table.max_tokens if torch.cuda.is_current_stream_capturing() else self.table.bound
        a.cells, a.len_bound, a.scaling = self._layer(layer), bound, scaling
        a.query, a.out, a.workspace = query.data_ptr(), out.data_ptr(), workspace.data_ptr()
        if key is not None:
            a.key, a.value, a.slots = key.data_ptr(), value.data_ptr(), self._slots.data_ptr()
        _lib.launch("dkv_q4_attend", a, self.device)
        return out

    def begin(self, counts=None) -> None:
        """How many tokens of every row the next forward pass brings (int32 [n_seq] or a list): rows are padded at
        their end. Without it, every row is full."""
        self._counts = counts if counts is None else self.table._counts(counts)

    def attend(self, module, query, key, value, attention_mask, scaling):
        """Same contract as an HF attention function: (output, None). The pass's first layer plans its tokens. A
        mask [rows or 1, any heads, q_len, q_len or more] may only repeat the causal order: of its columns the last q_len
        are the new tokens, those before them held ones, which every new token sees. Another one is refused through the
        status word."""
        q_len = query.shape[2]
        if key.shape[2] != q_len:
            raise ValueError(f"{key.shape[2]} keys for {q_len} queries: pass the batch's own cache (Q4Batch.cache) to "
                             "the model")
        if attention_mask is not None:
            form = tuple(attention_mask.shape)
            if len(form) != 4 or form[0] not in (1, self.n_seq) or form[2] != q_len or form[3] < q_len:
                raise ValueError(f"a mask {form} is not [1 or {self.n_seq}, heads, {q_len}, {q_len} or more]")
            if attention_mask.device != self.device:
                raise ValueError(f"the mask is on {attention_mask.device}, the cache on {self.device}")
        if module.layer_idx == 0:
            # what attend_layer would refuse is refused before the tokens have their places
            self._check("query", query, self.q_heads, q_len)
            self._check("key", key, self.kv_heads, q_len)
            self._check("value", value, self.kv_heads, q_len)
            counts, self._counts = self._counts, None
            self.plan(counts, q_len)
            if attention_mask is not None:
                self._check_mask(attention_mask, counts, q_len)
        out_dtype = torch.promote_types(query.dtype, self.dtype)
        return self.attend_layer(module.layer_idx, query, key, value, scaling, out_dtype=out_dtype), None

    def _check_mask(self, mask: torch.Tensor, counts, q_len: int) -> None:
        visible = mask if mask.dtype == torch.bool else mask == 0
        held = visible.shape[3] - q_len
        order = torch.ones(q_len, q_len, dtype=torch.bool, device=self.device).tril()
        wrong, hidden = visible[..., held:] != order, ~visible[..., :held]
        if counts is not None:
            real = torch.arange(q_len, device=self.device) < counts[:, None]
            wrong = wrong & real[:, None, :, None] & real[:, None, None, :]
            hidden = hidden & real[:, None, :, None]
        self.status.masked_fill_((wrong.any() | hidden.any()) & (self.status == 0), MASK_ERROR)

    # ------------------------------------------------------------------ status
    @property
    def poll_wait_s(self) -> float:
        return self.table.poll_wait_s

    @poll_wait_s.setter
    def poll_wait_s(self, seconds: float) -> None:
        self.table.poll_wait_s = seconds

    def check_status(self) -> None:
        self.table.check_status()

    def poll_status(self, depth: int | None = None) -> None:
        """Bounded per-step check of the status word, as ``CompressedBatch.poll_status``."""
        self.table.poll_status(depth)

    def reset_status(self) -> None:
        """Clear a recorded device error; until then the kernels do no work."""
        self.table.reset_status()


class Q4Context:
    """A prefilled conversation in 4 bits, attended to directly: ``greedy_answer(model, tokenizer, context,
    context.exact_cache, ...)`` as with ``CompressedContext``. ``keys`` / ``values`` per layer
    [1, kv_heads, tokens, head_dim]; ``room`` tokens can follow."""

    def __init__(self, keys: list[torch.Tensor], values: list[torch.Tensor], model, dtype=torch.float16, room: int = 1024):
        _, heads, tokens, dim = keys[0].shape
        self.model, self.dtype, self.context_tokens = model, dtype, tokens
        self.batch = Q4Batch(1, layers=len(keys), kv_heads=heads, q_heads=model.config.num_attention_heads,
                             head_dim=dim, max_tokens=tokens + room, device=keys[0].device, dtype=dtype)
        self.batch.plan(None, tokens)
        for layer, (k, v) in enumerate(zip(keys, values)):
            self.batch.append(layer, k, v)
        self.exact_cache = self.batch.cache

    def code_bytes(self) -> int:
        """Bytes of the context's tokens in 4 bits."""
        return self.context_tokens * self.batch.token_bytes()

    def basis_bytes(self) -> int:
        return 0

    def exact_bytes(self) -> int:
        return 0

    def check_status(self) -> None:
        self.batch.check_status()

    def attend(self, module, query, key, value, attention_mask, scaling):
        return self.batch.attend(module, query, key, value, attention_mask, scaling)


def restore(keys: list[torch.Tensor], values: list[torch.Tensor]):
    """Per-layer [1, kv_heads, tokens, head_dim] -> the same through 4 bits (the cache that ``Methods.apply("q4")``
    rebuilds). 16-bit CUDA tensors go through the cells; others through ``quantise4``. A key or value that is not
    finite or beyond 2^15 raises ``DimmerKVError``."""
    if keys[0].is_cuda and keys[0].dtype in (torch.bfloat16, torch.float16):
        _, heads, tokens, dim = keys[0].shape
        batch = Q4Batch(1, layers=1, kv_heads=heads, q_heads=heads, head_dim=dim, max_tokens=max(1, tokens),
                        device=keys[0].device, dtype=keys[0].dtype)
        batch.plan(None, tokens)
        out = []
        for k, v in zip(keys, values):
            batch.append(0, k, v)
            out.append(batch.read(0))
        batch.check_status()
        return [k for k, _ in out], [v for _, v in out]
    def through(x):
        if x.numel() and not bool((x.abs() <= CELL_MAX).all()):  # (false for a NaN)
            raise _lib.DimmerKVError(_lib.describe_device_error(CELL_ERROR))
        return dequantise4(*quantise4(x)).to(x.dtype)

    return [through(k) for k in keys], [through(v) for v in values]
