"""Block tables of a paged cache, kept and changed on the GPU.

``PageTable`` holds, for a batch of conversations, which pages of a shared pool hold their tokens, how many tokens
they have and which pages are free. ``plan`` makes room for new tokens and returns the slot of each; ``trim`` keeps
the first tokens of every conversation and gives the other pages back (a rejected draft, or a finished
conversation with 0). Counts and lengths are device tensors and nothing is read back, so a step can be captured
into a CUDA graph. A failed plan changes nothing: its slots are -1 and the status word tells (``poll_status``).
"""

from __future__ import annotations

import torch

from . import _lib

PAGE = 64  # tokens of a page (DKV_PAGE_TOKENS)
MAX_SEQ = 8192


def pages_of(tokens: int) -> int:
    return -(-tokens // PAGE)


class PageTable:
    """Pages of ``n_seq`` conversations of up to ``max_tokens`` tokens out of a pool of ``n_pages``.

    ``blocks`` int32 [n_seq, max_blocks] the pages in token order (-1: none), ``lengths`` int32 [n_seq] the tokens,
    ``starts`` int32 [n_seq] the tokens before the newest plan. ``free`` (optional, int32 [n]) gives the free
    pages, each once, the last one taken first; default: all, page 0 first."""

    def __init__(self, n_seq: int, n_pages: int, max_tokens: int, device="cuda", free: torch.Tensor | None = None,
                 status: torch.Tensor | None = None):
        if not 1 <= n_seq <= MAX_SEQ:
            raise ValueError(f"{n_seq} conversations: a table holds 1 to {MAX_SEQ}")
        if max_tokens < 1 or n_pages < 1:
            raise ValueError("max_tokens and n_pages must be at least 1")
        if max(n_pages, pages_of(max_tokens)) * PAGE > 2**31 - 1:
            raise ValueError("slots are 32-bit: at most 2^31 - 1 tokens in the pool and per conversation")
        if free is not None and (free.dtype != torch.int32 or free.dim() != 1 or free.numel() > n_pages):
            raise ValueError("free must be an int32 vector of at most n_pages pages")
        if free is not None and free.numel():
            pages = free.cpu()
            if int(pages.min()) < 0 or int(pages.max()) >= n_pages or int(pages.bincount().max()) > 1:
                raise ValueError(f"free must list pages of 0 .. {n_pages - 1}, each once")
        self.device = _lib.cuda_device(device)
        self.n_seq, self.n_pages, self.max_tokens = n_seq, n_pages, max_tokens
        self.max_blocks = pages_of(max_tokens)
        self.blocks = torch.full((n_seq, self.max_blocks), -1, dtype=torch.int32, device=self.device)
        self.lengths = torch.zeros(n_seq, dtype=torch.int32, device=self.device)
        self.starts = torch.zeros(n_seq, dtype=torch.int32, device=self.device)
        self.free = torch.empty(n_pages, dtype=torch.int32, device=self.device)
        given = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=self.device) if free is None else free
        self.free[:given.numel()] = given.to(self.device)
        self.n_free = torch.full((1,), given.numel(), dtype=torch.int32, device=self.device)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device) if status is None else status
        self.poll_wait_s = 60.0
        self._poller = None
        self.bound = 0  # no length is above this (known on the host), whatever replays of captured plans reach
        self._even: dict[int, torch.Tensor] = {}
        self._args = _lib.PageArgs(self.blocks.data_ptr(), self.max_blocks, self.lengths.data_ptr(),
                                   self.starts.data_ptr(), self.free.data_ptr(), self.n_free.data_ptr(), n_pages, n_seq,
                                   None, 0, None, self.status.data_ptr())

    def even(self, count: int) -> torch.Tensor:
        """int32 [n_seq] of ``count`` everywhere (kept: the same tensor for the same count)."""
        t = self._even.get(count)
        if t is None:
            t = torch.full((self.n_seq,), count, dtype=torch.int32, device=self.device)
            # one made in a capture is filled when the graph runs, and lives in the graph's memory
            if not torch.cuda.is_current_stream_capturing():
                self._even[count] = t
        return t

    def _counts(self, counts) -> torch.Tensor:
        if isinstance(counts, torch.Tensor):
            if counts.device != self.device or counts.dtype != torch.int32 or counts.shape != (self.n_seq,):
                raise ValueError(f"counts must be int32 [{self.n_seq}] on {self.device}")
            counts = counts.contiguous()
            # the kernels change these two while they read the counts
            if counts.data_ptr() in (self.lengths.data_ptr(), self.starts.data_ptr()):
                counts = counts.clone()
            return counts
        counts = [int(c) for c in counts]
        if len(counts) != self.n_seq:
            raise ValueError(f"{len(counts)} counts for {self.n_seq} conversations")
        return torch.tensor(counts, dtype=torch.int32, device=self.device)

    def _run(self, name: str, counts: torch.Tensor, q_len: int, slots: torch.Tensor | None) -> None:
        a = _lib.PageArgs.from_buffer_copy(self._args)
        a.counts, a.q_len = counts.data_ptr(), q_len
        if slots is not None:
            a.slots = slots.data_ptr()
        _lib.launch(name, a, self.device)

    def plan(self, counts=None, q_len: int = 1) -> torch.Tensor:
        """Room for ``counts[s]`` (0 .. q_len) more tokens of every conversation; ``None``: q_len each. Returns the
        slots int32 [n_seq, q_len] (page * 64 + place), -1 behind a conversation's new tokens."""
        if q_len < 0:
            raise ValueError("q_len must not be negative")
        counts = self.even(q_len) if counts is None else self._counts(counts)
        slots = torch.empty(self.n_seq, q_len, dtype=torch.int32, device=self.device)
        self._run("dkv_page_plan", counts, q_len, slots)
        # replays of a captured plan lengthen the conversations without passing here
        self.bound = self.max_tokens if torch.cuda.is_current_stream_capturing() else min(self.max_tokens, self.bound + q_len)
        return slots

    def trim(self, keep) -> None:
        """Keep the first min(length, keep[s]) tokens of every conversation and give the other pages back."""
        self._run("dkv_page_trim", self._counts(keep), 0, None)

    def slots(self, count: int) -> torch.Tensor:
        """The slots of the tokens 0 .. count - 1 of every conversation, int32 [n_seq, count], -1 where it has
        fewer."""
        if not 0 <= count <= self.max_tokens:
            raise ValueError(f"count must be 0 .. {self.max_tokens}")
        slots = torch.empty(self.n_seq, count, dtype=torch.int32, device=self.device)
        a = _lib.PageArgs.from_buffer_copy(self._args)
        counts = self.lengths.clamp(max=count)
        a.starts, a.counts, a.q_len, a.slots = self.even(0).data_ptr(), counts.data_ptr(), count, slots.data_ptr()
        _lib.launch("dkv_page_slots", a, self.device)
        return slots

    def check_status(self) -> None:
        _lib.check_device_status(self.status)

    def poll_status(self, depth: int | None = None) -> None:
        """Bounded per-step check of the status word (``_lib.StatusPoller``)."""
        if self._poller is None:
            self._poller = _lib.StatusPoller(self.status, depth=2, max_wait_s=self.poll_wait_s)
        self._poller.poll(depth)

    def reset_status(self) -> None:
        """Clear a recorded device error; until then the kernels do no work."""
        self.status.zero_()
