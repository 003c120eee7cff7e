"""Beam search, and greedy decoding of many rows behind a shared prefix (not in the reference).

Both keep the shared tokens once. ``generate_beam`` prefills each prompt into a
prefix cache of one row per prompt; its beams hold only their new tokens. A
step is one forward of all beams (``ops.shared_prefix_attention`` in every
layer), the selection over beams and vocabulary (``VocabParallelLMHead.beam_select``)
and the reordering of the beams' caches (``KVCache.reorder_``).
``generate_shared_prefix`` runs rows with prompts of their own behind one (or a
few) shared prompts.

At tp = 1 the step is captured into a CUDA graph once per shape and replayed,
as ``generate_greedy`` does; its state (tokens, scores, cursors) lives on the
device. With tp > 1 the exchange of candidates goes through torch.distributed
and the steps run without a graph.
"""

from __future__ import annotations

import torch

from minitp_b200 import _lib
from minitp_b200.generation import make_kv_cache, select_token
from minitp_b200.layer import TPQwen2ForCausalLM


_MAX_SHARED_SESSIONS = 4


class _SharedSession:
    """Buffers of one shape behind a shared prefix, and the CUDA graph of its step.

    Kept on the model between calls, apart from the greedy decode sessions (these
    keep their places whatever shapes are searched), and dropped with the native
    model. ``slot`` and ``rope`` are the new token's place in the own
    cache and its position; ``lens`` the own cache's length after it, per row.
    """

    def __init__(self, model: TPQwen2ForCausalLM, native: int, groups: int, width: int, prefix: int, cap: int,
                 new: int, device: torch.device) -> None:
        n = groups * width
        self.native = native
        self.prefix = make_kv_cache(model, groups, prefix)
        self.own = make_kv_cache(model, n, max(1, cap))
        vloc = model.lm_head.vocab_end - model.lm_head.vocab_start
        self.logits = torch.empty(n, vloc, dtype=self.own.k[0].dtype, device=device)
        self.tok = torch.zeros(n, 1, dtype=torch.int64, device=device)
        self.slot = torch.zeros(1, dtype=torch.int32, device=device)
        self.rope = torch.zeros(1, dtype=torch.int64, device=device)
        self.lens = torch.zeros(n, dtype=torch.int32, device=device)
        self.at = torch.zeros(1, dtype=torch.int64, device=device)  # column of `seqs` that the step writes
        self.seqs = torch.zeros(groups, width, new, dtype=torch.int64, device=device)
        self.scores = torch.zeros(groups, width, dtype=torch.float32, device=device)
        self.finished = torch.zeros(groups, width, dtype=torch.bool, device=device)
        self.graph: torch.cuda.CUDAGraph | None = None
        self.graph_epoch = -1

    def start(self, slot: int) -> None:
        """The first step puts its token at ``slot`` of the own cache."""
        self.slot.fill_(slot)
        self.rope.fill_(self.prefix.seq_len + slot)
        self.lens.fill_(slot + 1)
        self.at.fill_(1)

    def advance(self) -> None:
        for t in (self.slot, self.rope, self.lens, self.at):
            t.add_(1)

    def forward(self, model: TPQwen2ForCausalLM) -> None:
        model._forward_shared(self.tok, self.rope, self.own, self.slot, self.prefix, self.logits)

    def run(self, model: TPQwen2ForCausalLM, step, steps: int, done) -> int:
        """``step()`` up to ``steps`` times, until ``done()``; returns how often. The first call of a session
        runs eagerly (allocations, validation), later ones replay its graph."""
        graphs = model.ctx.tp_size == 1
        if self.graph is not None and self.graph_epoch != _lib.load().mtpb_settings_epoch():
            self.graph = None
        for i in range(steps):
            if done():
                return i
            if graphs and self.graph is not None:
                self.graph.replay()
                continue
            step()
            if graphs and i + 1 < steps:
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    step()
                self.graph, self.graph_epoch = g, _lib.load().mtpb_settings_epoch()
        return steps


def _session(model: TPQwen2ForCausalLM, kind: tuple, *shape) -> _SharedSession:
    """The model's session of this kind and shape (created on first use; at most four kept)."""
    native = model.native()  # first: (re)building the native model drops the model's sessions
    cache = model.__dict__.setdefault("_shared_sessions", {})
    key = (*kind, *(str(x) for x in shape))
    s = cache.pop(key, None)
    if s is None or s.native != native:
        s = _SharedSession(model, native, *shape)
    cache[key] = s
    while len(cache) > _MAX_SHARED_SESSIONS:
        cache.pop(next(iter(cache)))
    return s


def _check_positions(model: TPQwen2ForCausalLM, last: int) -> None:
    """The position table covers ``last`` tokens (a step on the device could only flag one behind it)."""
    if last > model.cfg.max_position_embeddings:
        raise ValueError(f"{last} positions needed, the model has {model.cfg.max_position_embeddings}")


@torch.inference_mode()
def generate_beam(
    model: TPQwen2ForCausalLM,
    input_ids: torch.Tensor,
    max_new_tokens: int,
    num_beams: int,
    eos_token_id: int | None = None,
    length_penalty: float = 0.0,
    num_return: int = 1,
    early_stop: bool = True,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Beam search: the ``num_return`` best continuations of each prompt, best first.

    ``input_ids [B, P]``. A hypothesis scores the sum of its tokens'
    log-probabilities. One that emitted ``eos_token_id`` keeps its score, competes
    with the others and repeats that token; with ``early_stop`` the search ends
    when every beam has. The result is ordered by score / length ** length_penalty
    (length: generated tokens up to the end token; 0: by the sum).

    Returns ``(ids [B, num_return, P + generated], scores [B, num_return])``, with
    the scores as ordered by.
    """
    if input_ids.dim() != 2 or input_ids.shape[1] < 1:
        raise ValueError(f"input_ids must be [B, P] with P >= 1, got {tuple(input_ids.shape)}")
    if not 1 <= num_beams <= 64 or not 1 <= num_return <= num_beams:
        raise ValueError(f"need 1 <= num_return <= num_beams <= 64, got {num_return} and {num_beams}")
    if max_new_tokens < 1:
        raise ValueError("max_new_tokens must be at least 1")
    if eos_token_id is not None and not 0 <= eos_token_id < model.cfg.vocab_size:
        raise ValueError(f"eos_token_id {eos_token_id} outside the vocabulary")
    b, p = input_ids.shape
    w, eos, head = num_beams, eos_token_id, model.lm_head
    _check_positions(model, p + max_new_tokens - 1)
    s = _session(model, ("beam", eos), b, w, p, max_new_tokens - 1, max_new_tokens, input_ids.device)
    s.prefix.seq_len = 0
    logits = model(input_ids, kv_cache=s.prefix, last_only=True)
    # the prompt is one live beam: its w best tokens start the search
    zero = torch.zeros(b, 1, dtype=torch.float32, device=input_ids.device)
    scores, _, tok, done = head.beam_select(logits, zero, w, None, eos)
    s.scores.copy_(scores)
    s.seqs.fill_(0 if eos is None else eos)
    s.seqs[:, :, 0] = tok
    s.tok.copy_(tok.view(b * w, 1))
    if eos is not None:
        s.finished.copy_(done)
    s.start(0)

    def step() -> None:
        s.forward(model)
        scores, parents, tok, done = head.beam_select(s.logits.view(b, w, -1), s.scores, w,
                                                      None if eos is None else s.finished, eos)
        s.own.reorder_(parents, s.lens)
        s.seqs.copy_(s.seqs.gather(1, parents[:, :, None].expand_as(s.seqs)))
        s.seqs.scatter_(2, s.at.expand(b, w, 1), tok[:, :, None])
        s.scores.copy_(scores)
        s.tok.copy_(tok.view(b * w, 1))
        if eos is not None:
            s.finished.copy_(done)
        s.advance()

    stops = early_stop and eos is not None
    ran = s.run(model, step, max_new_tokens - 1, lambda: stops and bool(s.finished.all()))
    seqs, scores = s.seqs[:, :, : ran + 1], s.scores
    if length_penalty != 0.0:
        length = torch.full_like(scores, ran + 1)
        if eos is not None:
            length = ((seqs != eos).sum(-1) + s.finished).to(scores.dtype)
        scores = scores / length ** length_penalty
    scores, order = scores.sort(dim=1, descending=True, stable=True)
    seqs = seqs.gather(1, order[:, :, None].expand_as(seqs))
    prompt = input_ids.to(torch.int64)[:, None].expand(b, num_return, p)
    return torch.cat([prompt, seqs[:, :num_return]], -1), scores[:, :num_return].clone()


@torch.inference_mode()
def generate_shared_prefix(
    model: TPQwen2ForCausalLM,
    prefix_ids: torch.Tensor,
    input_ids: torch.Tensor,
    max_new_tokens: int,
    eos_token_id: int | None = None,
    early_stop: bool = True,
) -> torch.Tensor:
    """Greedy decode of rows whose prompts start with the same tokens; the shared part is kept and prefilled once.

    ``prefix_ids [G, P]``; ``input_ids [N, T]``, N / G consecutive rows to a
    prefix. Row n continues ``prefix_ids[n // (N / G)]`` followed by
    ``input_ids[n]``. Returns ``[N, T + generated]`` (without the prefix), as
    ``generate_greedy`` returns its rows.
    """
    if prefix_ids.dim() != 2 or input_ids.dim() != 2 or prefix_ids.shape[1] < 1 or input_ids.shape[1] < 1:
        raise ValueError("prefix_ids and input_ids must be [G, P] and [N, T], with tokens")
    g, p = prefix_ids.shape
    n, t = input_ids.shape
    if g < 1 or n < g or n % g:
        raise ValueError(f"{n} rows do not divide into {g} shared prefixes")
    if max_new_tokens < 1:
        raise ValueError("max_new_tokens must be at least 1")
    _check_positions(model, p + t + max_new_tokens - 1)
    stops = early_stop and eos_token_id is not None
    eos = eos_token_id if stops else None
    s = _session(model, ("prefix", eos), g, n // g, p, t + max_new_tokens - 1, max_new_tokens, input_ids.device)
    s.prefix.seq_len = s.own.seq_len = 0
    model(prefix_ids, kv_cache=s.prefix, last_only=True)
    logits = model(input_ids, kv_cache=s.own, last_only=True, prefix_cache=s.prefix)
    tok = select_token(model, logits)
    rows = s.seqs.view(n, max_new_tokens)
    rows[:, 0] = tok
    s.tok.copy_(tok[:, None])
    flags = s.finished.view(n)
    if stops:
        flags.copy_(tok == eos)
    s.start(t)

    def step() -> None:
        s.forward(model)
        tok = select_token(model, s.logits[:, None])
        if stops:
            tok = torch.where(flags, eos, tok)
            flags.logical_or_(tok == eos)
        rows.scatter_(1, s.at.expand(n, 1), tok[:, None])
        s.tok.copy_(tok[:, None])
        s.advance()

    ran = s.run(model, step, max_new_tokens - 1, lambda: stops and bool(flags.all()))
    return torch.cat([input_ids.to(torch.int64), rows[:, : ran + 1]], -1)


__all__ = ["generate_beam", "generate_shared_prefix"]
