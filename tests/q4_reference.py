"""The paged 4-bit cache's operators in plain operations of 64 bits, for the tests."""

from __future__ import annotations

import math

import numpy as np
import torch

GROUP = 64
PAGE = 64


def half(x: torch.Tensor) -> torch.Tensor:
    return x.float().half().double()


def cells64(x: torch.Tensor):
    """(values, scales, lows) in float64 that 4 bits hold for x [..., dim]; scales / lows [..., dim / 64]."""
    g = x.double().unflatten(-1, (-1, GROUP))
    low = half(g.amin(-1))
    scale = half(((g.amax(-1) - low).float() / 15.0))
    step = scale[..., None]
    code = torch.where(step > 0, ((g - low[..., None]) / step.clamp_min(1e-30)).round().clamp(0, 15), 0.0)
    return (low[..., None] + code * step).flatten(-2), scale, low


def attend64(query, key, value, held, scaling):
    """One conversation: query [hq, n, d] of the tokens held .. held + n - 1 over key / value [hkv, held + n, d]
    (16-bit tensors). Returns the output [n, hq, d] in float64 and what attend_tolerance goes by: the sums of
    p * scale * code and of p * |low| per output, the largest sum of a score's absolute terms per row, the number of
    tokens and the largest value scale."""
    hq, n, d = query.shape
    share = hq // key.shape[0]
    k, ks, kl = (t.repeat_interleave(share, 0) for t in cells64(key))
    v, vs, vl = (t.repeat_interleave(share, 0) for t in cells64(value))
    vl = vl.repeat_interleave(GROUP, -1)
    q = query.double()
    scores = q @ k.transpose(1, 2) * scaling
    hidden = torch.arange(k.shape[1], device=q.device) > held + torch.arange(n, device=q.device)[:, None]
    p = torch.softmax(scores.masked_fill(hidden, -math.inf), -1)
    width = (15 * ks + kl.abs()).repeat_interleave(GROUP, -1)
    terms = (q.abs() @ width.transpose(1, 2) * scaling).masked_fill(hidden, 0.0).amax(-1)
    parts = (p @ (v - vl)).transpose(0, 1), (p @ vl.abs()).transpose(0, 1), terms.transpose(0, 1), k.shape[1], float(vs.max())
    return (p @ v).transpose(0, 1), parts


def attend_tolerance(out, parts, dtype, out_dtype, rows=1):
    """Largest error of dkv_q4_attend against attend64, for a cache of ``dtype`` and ``rows`` query rows per KV head.

    Up to 64 rows: p * scale is rounded to float16 (half a step: 2^-11) in front of its code, or, for float16 caches, to
    two float16 numbers (2^-21 between them): that much of the sum of p * scale * code. Below 2^-14 the half step is
    2^-25 instead, of p * 2^7 * scale / 2^k with 2^k at most 4 times the largest scale, times a code of at most 15:
    2^-26 of the largest scale for every token.
    More rows: keys, values and probabilities are rounded to float16, for float16 caches keys and values to two
    numbers: a score moves by 2^-11 (2^-21) of its absolute terms, numerator and denominator by that; the sum by 2^-11
    for the probabilities and 2^-11 (2^-21) for the values, and a probability below 2^-14 of 2^7 by 2^-32 of the
    largest value (15 scales and a low) for every token.
    A score, a float32 sum of absolute terms ``terms`` in at most 2 * 128 additions whose operands the tensor core may
    cut at 2^-22, is off by at most 2^-17 of them in all, which moves numerator and denominator by that much each. The
    float32 sums over tokens, chains of at most four products that the tensor core may cut at 2^-22 each and float32
    additions of their sums, a few hundred per warp, are good to 2^-16 of their absolute terms (the longer chains of
    more rows, over values of either sign, to 2^-14). The output is rounded once, to half a step of its type."""
    coded, low, terms, tokens, scale = parts
    step = 2**-11 if dtype == torch.bfloat16 else 2**-21
    if rows <= 64:
        own = coded * step + (coded + low) * 2**-16 + tokens * 2**-26 * scale
    else:
        own = (coded + low) * (2**-11 + step + 2 * step * terms[..., None] + 2**-14) + tokens * 2**-32 * 32 * scale
    return own + (coded + low) * 2 * 2**-17 * terms[..., None] + out.abs() * torch.finfo(out_dtype).eps / 2 + 1e-12


class PlainTable:
    """PageTable in plain Python."""

    def __init__(self, n_seq, n_pages, max_tokens):
        self.free = list(range(n_pages - 1, -1, -1))
        self.blocks = [[] for _ in range(n_seq)]
        self.lengths = [0] * n_seq
        self.starts = [0] * n_seq
        self.cols = -(-max_tokens // PAGE)

    def plan(self, counts, q_len):
        slots = np.full((len(counts), q_len), -1, dtype=np.int32)
        for s, c in enumerate(counts):
            self.starts[s] = self.lengths[s]
            for i in range(c):
                at = self.lengths[s] + i
                if at // PAGE == len(self.blocks[s]):
                    self.blocks[s].append(self.free.pop())
                slots[s, i] = self.blocks[s][at // PAGE] * PAGE + at % PAGE
            self.lengths[s] += c
        return slots

    def trim(self, keep):
        back = []
        for s, k in enumerate(keep):
            self.lengths[s] = self.starts[s] = min(self.lengths[s], k)
            held = -(-self.lengths[s] // PAGE)
            back += self.blocks[s][held:]
            del self.blocks[s][held:]
        self.free += back[::-1]

    def array(self):
        out = np.full((len(self.blocks), self.cols), -1, dtype=np.int32)
        for s, row in enumerate(self.blocks):
            out[s, :len(row)] = row
        return out


def rules64(logits, history, lengths, prompts, repetition, frequency, presence, bias=None, allowed=None):
    """Adjusted logits in float64 [rows, vocab] from lists / arrays on the host."""
    x = logits.double().cpu().clone()
    for r in range(x.shape[0]):
        ids = [int(t) for t in history[r][:lengths[r]]]
        for t in sorted({t for t in ids if 0 <= t < x.shape[1]}):
            made = sum(1 for u in ids[prompts[r]:] if u == t)
            v = float(x[r, t])
            v = v / repetition[r] if v > 0 else v * repetition[r]
            if made:
                v = v - frequency[r] * made - presence[r]
            x[r, t] = v
        if bias is not None:
            for t, b in zip(bias[0][r], bias[1][r]):
                if 0 <= int(t) < x.shape[1]:
                    x[r, int(t)] += float(b)
        if allowed is not None:
            for t in range(x.shape[1]):
                if not (int(allowed[r, t // 32]) >> (t % 32)) & 1:
                    x[r, t] = -math.inf
    return x
