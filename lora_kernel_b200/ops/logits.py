"""Logits before sampling: penalties for tokens already seen, biases, grammar
masks, and the table of token counts that the penalties read.

counts is int16 [rows, vocab], a row per running request: bit 15 says that the
token is in the prompt, bits 0-14 how often it was generated (up to 32767).
"""
from __future__ import annotations

from typing import Dict, Optional, Sequence, Tuple

import torch

from .._ext import C, require_device, status


def token_counts(rows: int, vocab: int, device="cuda") -> torch.Tensor:
    """An empty table of token counts (rows padded to 16 bytes: a view of a wider table where vocab is odd)."""
    return torch.zeros(rows, (vocab + 7) // 8 * 8, dtype=torch.int16, device=device)[:, :vocab]


def set_token_counts(counts: torch.Tensor, rows: Optional[torch.Tensor], tokens: torch.Tensor, offsets: torch.Tensor,
                     prompt_lens: torch.Tensor) -> None:
    """Write the rows of n requests from their histories (admission, readmission).

    tokens int64: the histories one after another, history i at
    tokens[offsets[i]:offsets[i + 1]] (int32 [n + 1]), its first prompt_lens[i]
    tokens the prompt.  rows int32 [n]: the request's row (None: row i;
    negative: skip)."""
    require_device(counts)
    C().set_token_counts(counts, rows, tokens, offsets, prompt_lens, status(counts.device))


def add_token_counts(counts: torch.Tensor, rows: Optional[torch.Tensor], tokens: torch.Tensor) -> None:
    """Count generated tokens int64 [n], token i in row rows[i] (int32; None: row i; negative: skip)."""
    require_device(counts)
    C().add_token_counts(counts, rows, tokens, status(counts.device))


def logit_bias(biases: Sequence[Optional[Dict[int, float]]], device="cuda") -> Optional[Tuple[torch.Tensor, ...]]:
    """(offsets, ids, values) of each row's {token id: bias} (None or {} where a row has none)."""
    if not any(biases):
        return None
    offsets, ids, values = [0], [], []
    for b in biases:
        for k, v in (b or {}).items():
            ids.append(int(k))
            values.append(float(v))
        offsets.append(len(ids))
    return (torch.tensor(offsets, dtype=torch.int32, device=device), torch.tensor(ids, dtype=torch.int32, device=device),
            torch.tensor(values, dtype=torch.float32, device=device))


def adjust_logits(logits: torch.Tensor, counts: Optional[torch.Tensor] = None, rows: Optional[torch.Tensor] = None,
                  penalties: Optional[torch.Tensor] = None, *, bias: Optional[Tuple[torch.Tensor, ...]] = None,
                  mask: Optional[torch.Tensor] = None, mask_rows: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """logits [n, vocab] (bf16 or fp32) -> the adjusted logits (out may be logits).

    For a token that row rows[i] of counts has seen: z / r where z > 0, else
    z * r (repetition); then z - frequency * count - presence * [count > 0],
    count being how often it was generated; penalties fp32 [n, 3] holds
    (repetition, frequency, presence).  rows int32 [n]: None = row i, negative
    = no penalties.  Then bias (offsets int32 [n + 1], ids int32, values fp32)
    is added (an id named more than once: its values' sum, in the list's order),
    and tokens whose bit in mask int32 [m, ceil(vocab / 32)] is 0
    become -inf; mask_rows int32 [n]: None = row i, negative = unrestricted.
    fp32 throughout, rounded once."""
    require_device(logits)
    o, i, v = bias if bias is not None else (None, None, None)
    return C().adjust_logits(logits, counts, rows, penalties, o, i, v, mask, mask_rows, out, status(logits.device))
