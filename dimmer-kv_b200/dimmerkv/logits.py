"""Rules on the logits of a decode step: penalties for repeated tokens, biases, a grammar mask, and the choice.

``LogitRules`` holds, for every row of a batch, the tokens so far (on the GPU) and the row's penalties and biases.
``apply`` returns the adjusted logits and the best token; ``pick`` returns the token and appends it to the row's
history on the device, so a captured step needs no host in between. ``greedy_answer`` and
``greedy_decode_batch`` take a ``LogitRules`` as ``rules``.
"""

from __future__ import annotations

import torch

from . import _lib

MAX_BIAS = 1024
DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def allow_mask(tokens: list, vocab: int, device="cuda") -> torch.Tensor:
    """Bit mask int32 [rows, ceil(vocab / 32)] that allows, in row r, the tokens ``tokens[r]`` and no other."""
    allowed = torch.zeros(len(tokens), (vocab + 31) // 32 * 32, dtype=torch.int64)
    for r, row in enumerate(tokens):
        ids = torch.as_tensor(list(row), dtype=torch.int64)
        if ids.numel() and (int(ids.min()) < 0 or int(ids.max()) >= vocab):
            raise ValueError(f"row {r} allows tokens outside 0 .. {vocab - 1}")
        allowed[r, ids] = 1
    words = (allowed.view(len(tokens), -1, 32) << torch.arange(32)).sum(-1)
    return torch.where(words >= 2**31, words - 2**32, words).to(torch.int32).to(device)


class LogitRules:
    """Rules of ``n_rows`` rows over ``vocab`` tokens, with room for ``capacity`` tokens of history per row.

    For a token seen in the history x becomes x / repetition where positive, x * repetition elsewhere; for one
    generated c > 0 times x - frequency * c - presence; ``bias_values`` are added at ``bias_ids`` (int32 [n_rows, n],
    -1: none; listed twice: their sum); where the mask does not allow a token it is -infinity. Penalties are numbers
    or float32 [n_rows] tensors; a repetition must be above 0."""

    def __init__(self, n_rows: int, vocab: int, device="cuda", capacity: int = 4096, repetition=1.0, frequency=0.0,
                 presence=0.0, bias_ids: torch.Tensor | None = None, bias_values: torch.Tensor | None = None):
        if n_rows < 1 or vocab < 1 or capacity < 1:
            raise ValueError("n_rows, vocab and capacity must be at least 1")
        if not isinstance(repetition, torch.Tensor) and not repetition > 0:
            raise ValueError("repetition must be above 0")
        if (bias_ids is None) != (bias_values is None):
            raise ValueError("bias_ids and bias_values come together")
        if bias_ids is not None and (bias_ids.shape != bias_values.shape or bias_ids.dim() != 2 or
                                     bias_ids.shape[0] != n_rows or bias_ids.shape[1] > MAX_BIAS):
            raise ValueError(f"bias_ids and bias_values must be [{n_rows}, n] with n at most {MAX_BIAS}")
        for name, p in (("repetition", repetition), ("frequency", frequency), ("presence", presence)):
            if isinstance(p, torch.Tensor) and p.shape != (n_rows,):
                raise ValueError(f"{name} must be a number or [{n_rows}]")
        self.device = _lib.cuda_device(device)
        self.n_rows, self.vocab, self.capacity = n_rows, vocab, capacity
        self.history = torch.full((n_rows, capacity), -1, dtype=torch.int32, device=self.device)
        self.lengths = torch.zeros(n_rows, dtype=torch.int32, device=self.device)
        self.prompts = torch.zeros(n_rows, dtype=torch.int32, device=self.device)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._held = [self._row(p) for p in (repetition, frequency, presence)]
        a = self._args = _lib.LogitsArgs()
        a.n_rows, a.vocab, a.capacity = n_rows, vocab, capacity
        a.history, a.lengths, a.prompts = self.history.data_ptr(), self.lengths.data_ptr(), self.prompts.data_ptr()
        a.repetition, a.frequency, a.presence = (t.data_ptr() for t in self._held)
        if bias_ids is not None and bias_ids.shape[1]:
            ids = bias_ids.to(device=self.device, dtype=torch.int32).contiguous()
            values = bias_values.to(device=self.device, dtype=torch.float32).contiguous()
            self._held += [ids, values]
            a.bias_ids, a.bias_values, a.n_bias = ids.data_ptr(), values.data_ptr(), ids.shape[1]
        a.status = self.status.data_ptr()

    def _row(self, p) -> torch.Tensor:
        if isinstance(p, torch.Tensor):
            return p.to(device=self.device, dtype=torch.float32).contiguous()
        return torch.full((self.n_rows,), float(p), dtype=torch.float32, device=self.device)

    def load(self, history: torch.Tensor, lengths=None, prompts=None) -> None:
        """The tokens so far: ``history`` [n_rows, n], of which row r has ``lengths[r]`` (default: all n), the first
        ``prompts[r]`` of them its prompt (default: all), the others generated."""
        n = history.shape[-1]
        if history.dim() != 2 or history.shape[0] != self.n_rows or n > self.capacity:
            raise ValueError(f"history must be [{self.n_rows}, at most {self.capacity}]")
        self.history[:, :n] = history.to(self.history)
        full = torch.full((self.n_rows,), n, dtype=torch.int32, device=self.device)
        self.lengths.copy_(full if lengths is None else torch.as_tensor(lengths, device=self.device).clamp(0, n))
        self.prompts.copy_(self.lengths if prompts is None else torch.as_tensor(prompts, device=self.device))

    def _run(self, logits: torch.Tensor, allowed: torch.Tensor | None, adjusted: bool, append: bool):
        if logits.shape != (self.n_rows, self.vocab):
            raise ValueError(f"logits {tuple(logits.shape)} are not [{self.n_rows}, {self.vocab}]")
        if logits.dtype not in DTYPES:
            raise ValueError(f"logits of {logits.dtype}: bfloat16, float16 or float32")
        if logits.device != self.device:
            raise ValueError(f"logits are on {logits.device}, the rules on {self.device}")
        if logits.stride(1) != 1 or logits.stride(0) < 0:
            logits = logits.contiguous()
        a = _lib.LogitsArgs.from_buffer_copy(self._args)
        if allowed is not None:
            words = (self.vocab + 31) // 32
            if allowed.dtype != torch.int32 or allowed.shape != (self.n_rows, words) or allowed.device != self.device:
                raise ValueError(f"allowed must be int32 [{self.n_rows}, {words}] on {self.device}")
            allowed = allowed.contiguous()
            a.allowed = allowed.data_ptr()
        tokens = torch.empty(self.n_rows, dtype=torch.int64, device=self.device)
        out = torch.empty(self.n_rows, self.vocab, dtype=torch.float32, device=self.device) if adjusted else None
        a.logits, a.dtype, a.row_stride = logits.data_ptr(), DTYPES[logits.dtype], logits.stride(0)
        a.adjusted, a.tokens, a.append = out.data_ptr() if adjusted else None, tokens.data_ptr(), int(append)
        _lib.launch("dkv_logit_rules", a, self.device)
        return out, tokens

    def apply(self, logits: torch.Tensor, allowed: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """(adjusted logits float32 [n_rows, vocab], best token int64 [n_rows], the lowest of equal ones, -1 where the
        mask leaves nothing) of logits [n_rows, vocab]; the history stays as it is."""
        return self._run(logits, allowed, True, False)

    def pick(self, logits: torch.Tensor, allowed: torch.Tensor | None = None) -> torch.Tensor:
        """The best token of every row, int64 [n_rows], appended to the row's history (-1: nothing allowed, nothing
        appended). A full history is told in the status word."""
        return self._run(logits, allowed, False, True)[1]

    def check_status(self) -> None:
        _lib.check_device_status(self.status)

    def reset_status(self) -> None:
        self.status.zero_()
