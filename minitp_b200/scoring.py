"""Scoring of given prompts: log-probabilities, entropies and top alternatives of their tokens (not in the reference).

``score_prompts`` takes prompts of any lengths in one call. They are packed one
behind the other, without padding, and run through the model in one forward
(``TPQwen2ForCausalLM.forward_packed``, whose attention is ``ops.prompt_attention``);
the LM head and ``VocabParallelLMHead.token_logprobs`` then take the tokens in
pieces, so that no more than a few hundred megabytes of logits exist at once.
(The forward itself goes in chunks of what one AllReduce message of the
communicator holds, 8 MB of hidden states by default: 4681 tokens of the 0.5B
shape in bf16, 1170 of the 7B one.)
"""

from __future__ import annotations

import operator
from dataclasses import dataclass
from typing import Sequence

import torch

from minitp_b200 import _lib, ops
from minitp_b200.layer import TPQwen2ForCausalLM

_LOGITS_BYTES = 256 << 20  # of one piece
_PROMPTS = 1 << 16  # of one forward (empty ones add no tokens; the attention takes 2^20)


@dataclass
class PromptScores:
    """Of one prompt of n tokens: row i belongs to token i + 1, given the tokens before it.

    ``logprobs`` and ``entropy`` fp32 ``[n - 1]`` (natural units), ``top_logprobs``
    fp32 and ``top_ids`` int64 ``[n - 1, top]``, best first (None with ``top`` 0).
    """

    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor | None
    top_ids: torch.Tensor | None


@torch.inference_mode()
def score_prompts(
    model: TPQwen2ForCausalLM,
    prompts: Sequence[torch.Tensor | Sequence[int]],
    top: int = 0,
    max_tokens: int = 32768,
) -> list[PromptScores]:
    """Scores of every prompt's tokens, given the tokens before them.

    ``prompts``: token ids, each a sequence of ints or an integer tensor ``[n]``
    on any device; ids outside the vocabulary are refused, and a prompt of one
    token or none has empty scores. ``top``: likeliest alternatives per token (0 to
    64). Prompts are packed into forwards of at most ``max_tokens`` tokens (a longer
    prompt goes alone). The results are on the model's device, and complete: errors
    that a kernel can only report to the device's status words (a wait that ran
    out) raise here.
    """
    dev = model.model.embed_tokens.weight.device
    if not 0 <= top <= 64:
        raise ValueError(f"top must be 0 .. 64, got {top}")
    if max_tokens < 1:
        raise ValueError(f"max_tokens must be positive, got {max_tokens}")
    ids = [p if isinstance(p, torch.Tensor) else _id_tensor(p) for p in prompts]
    for p in ids:
        if p.dim() != 1 or p.dtype.is_floating_point or p.dtype.is_complex or p.dtype == torch.bool:
            raise ValueError(f"prompts must be integer sequences [n], got {p.dtype} {tuple(p.shape)}")
        if p.numel() > model.cfg.max_position_embeddings:
            raise ValueError(f"{p.numel()} positions needed, the model has {model.cfg.max_position_embeddings}")
    for where in {p.device for p in ids}:  # (one look at each device's ids)
        some = torch.cat([p.to(torch.int64) for p in ids if p.device == where])
        if some.numel() and not bool(((some >= 0) & (some < model.cfg.vocab_size)).all()):
            raise ValueError(f"token ids outside the vocabulary of {model.cfg.vocab_size}")
    comm = model.ctx.comm() if dev.type == "cuda" else None
    before = comm.status() if comm else 0  # (what earlier calls left there is theirs, but for a peer that is gone)
    out: list[PromptScores] = []
    at = 0
    while at < len(ids):
        end, tokens = at, 0
        while end < len(ids) and end - at < _PROMPTS and (end == at or tokens + ids[end].numel() <= max_tokens):
            tokens += ids[end].numel()
            end += 1
        out += _score_packed(model, [p.to(dev, torch.int64) for p in ids[at:end]], top)
        at = end
    if comm:
        ops.raise_on_scoring_error(dev)
        if comm.status() & (~before | _lib.STATUS_TIMEOUT):
            comm.raise_on_error()
    return out


def _id_tensor(prompt: Sequence[int]) -> torch.Tensor:
    try:  # (torch would cut 1.5 to 1)
        return torch.tensor([operator.index(i) for i in prompt], dtype=torch.int64)
    except (TypeError, ValueError, OverflowError, RuntimeError) as e:
        raise ValueError(f"prompts must be integer sequences [n]: {e}") from None


def _score_packed(model: TPQwen2ForCausalLM, prompts: list[torch.Tensor], top: int) -> list[PromptScores]:
    dev = model.model.embed_tokens.weight.device
    lengths = [p.numel() for p in prompts]
    n = sum(lengths)
    starts = [0]
    for k in lengths:
        starts.append(starts[-1] + k)
    scored = [max(0, k - 1) for k in lengths]
    if n == 0 or sum(scored) == 0:
        parts = [torch.empty(0, dtype=torch.float32, device=dev)] * 2
        if top:
            parts += [torch.empty(0, top, dtype=torch.float32, device=dev), torch.empty(0, top, dtype=torch.int64, device=dev)]
    else:
        packed = torch.cat(prompts)
        hidden = model.forward_packed(packed, torch.tensor(starts, dtype=torch.int32).to(dev))
        # every token but a prompt's last predicts the one behind it
        rows = torch.cat([torch.arange(a, a + k) for a, k in zip(starts, scored)]).to(dev)
        hidden, targets = hidden[rows], packed[rows + 1]
        # (pieces of the largest shard's logits: every rank takes the same ones, as each is an exchange)
        piece = max(1, _LOGITS_BYTES // (model.lm_head._max_local_vocab() * hidden.element_size()))
        got = []
        for i in range(0, rows.numel(), piece):
            logits = ops.linear(hidden[i:i + piece], model.lm_head.weight)
            got.append(model.lm_head.token_logprobs(logits, targets[i:i + piece], top))
        parts = [torch.cat(p) for p in zip(*(g[:4 if top else 2] for g in got))]
    split = [p.split(scored) for p in parts]
    if not top:
        split += [[None] * len(prompts)] * 2
    return [PromptScores(*row) for row in zip(*split)]


__all__ = ["PromptScores", "score_prompts"]
