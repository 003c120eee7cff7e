"""Tensor-level wrappers of the C ABI (include/minitp_b200.h).

Each function validates device, dtype and layout, allocates its outputs with
torch (device memory plumbing) and enqueues the kernel on the current CUDA
stream. None of them has a CPU path: CPU tensors raise.
"""

from __future__ import annotations

import array
import operator

import torch

from minitp_b200 import _lib


def _c(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.contiguous()


def _comm_handle(comm) -> int | None:
    return None if comm is None else comm.handle


def linear(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    """``F.linear(x, w, bias)`` on the weight-streaming GEMV (fp32 accumulate)."""
    _lib.require_cuda(x, w, bias)
    if x.dtype != w.dtype or (bias is not None and bias.dtype != w.dtype):
        raise _lib.MinitpB200Error(f"linear: dtype mismatch ({x.dtype}, {w.dtype})")
    n, k = w.shape
    if x.shape[-1] != k:
        raise _lib.MinitpB200Error(f"linear: x has {x.shape[-1]} features, weight expects {k}")
    x2 = _c(x).reshape(-1, k)
    m = x2.shape[0]
    y = torch.empty(*x.shape[:-1], n, dtype=x.dtype, device=x.device)
    if m == 0:
        return y
    w = _c(w)
    _lib.call("mtpb_linear", x2.data_ptr(), k, w.data_ptr(), _lib.ptr(None if bias is None else _c(bias)),
              y.data_ptr(), n, m, n, k, _lib.dtype_code(x.dtype), _lib.stream_ptr(x.device))
    return y


def linear_swiglu(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """``silu(gate) * up`` with ``gate, up = F.linear(x, w).chunk(2, -1)``."""
    _lib.require_cuda(x, w)
    n2, k = w.shape
    inter = n2 // 2
    x2 = _c(x).reshape(-1, k)
    m = x2.shape[0]
    y = torch.empty(*x.shape[:-1], inter, dtype=x.dtype, device=x.device)
    if m == 0:
        return y
    _lib.call("mtpb_linear_swiglu", x2.data_ptr(), k, _c(w).data_ptr(), y.data_ptr(), inter, m, inter, k,
              _lib.dtype_code(x.dtype), _lib.stream_ptr(x.device))
    return y


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    _lib.require_cuda(x, w)
    h = x.shape[-1]
    x2 = _c(x).reshape(-1, h)
    y = torch.empty_like(x2)
    if x2.shape[0]:
        _lib.call("mtpb_rmsnorm", x2.data_ptr(), _c(w).data_ptr(), y.data_ptr(), x2.shape[0], h, float(eps),
                  _lib.dtype_code(x.dtype), _lib.stream_ptr(x.device))
    return y.view(x.shape)


def allreduce_(t: torch.Tensor, comm) -> torch.Tensor:
    """In-place SUM over the communicator's ranks (one-shot NVLink push)."""
    _lib.require_cuda(t)
    if not t.is_contiguous():
        raise _lib.MinitpB200Error("allreduce_: tensor must be contiguous")
    h = t.shape[-1]
    _lib.call("mtpb_allreduce", _comm_handle(comm), t.data_ptr(), t.numel() // h, h, _lib.dtype_code(t.dtype),
              _lib.stream_ptr(t.device))
    return t


def allreduce_residual_rmsnorm(
    partial: torch.Tensor,
    residual: torch.Tensor | None,
    gain: torch.Tensor | None,
    eps: float,
    comm,
    bias: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """(residual + T(sum_r partial_r) [+ bias], RMSNorm of that) in one kernel."""
    _lib.require_cuda(partial, residual, gain, bias)
    h = partial.shape[-1]
    p = _c(partial)
    rows = p.numel() // h
    out_res = torch.empty_like(p)
    out_norm = torch.empty_like(p) if gain is not None else None
    if rows:
        _lib.call(
            "mtpb_allreduce_residual_rmsnorm", _comm_handle(comm), p.data_ptr(),
            _lib.ptr(None if residual is None else _c(residual)), _lib.ptr(None if gain is None else _c(gain)),
            _lib.ptr(None if bias is None else _c(bias)), out_res.data_ptr(), _lib.ptr(out_norm),
            rows, h, float(eps), _lib.dtype_code(p.dtype), _lib.stream_ptr(p.device),
        )
    return out_res, out_norm


def embedding(ids: torch.Tensor, table: torch.Tensor, vstart: int, vend: int, vocab: int, comm) -> torch.Tensor:
    """Masked local lookup of ``ids`` in the shard [vstart, vend), summed over ranks."""
    _lib.require_cuda(ids, table)
    ids2 = _c(ids.to(torch.int64)).reshape(-1)
    h = table.shape[1]
    out = torch.empty(*ids.shape, h, dtype=table.dtype, device=table.device)
    if ids2.numel():
        _lib.call("mtpb_embedding", _comm_handle(comm), ids2.data_ptr(), _c(table).data_ptr(), out.data_ptr(),
                  ids2.numel(), h, vstart, vend, vocab, _lib.dtype_code(table.dtype), _lib.stream_ptr(table.device))
    return out


def argmax(local_logits: torch.Tensor, vstart: int, comm) -> torch.Tensor:
    """Greedy ids over vocab-sharded logits ``[..., V_local]`` -> ``[..., 1]`` int64."""
    _lib.require_cuda(local_logits)
    v = local_logits.shape[-1]
    x = local_logits.reshape(-1, v)
    if x.stride(-1) != 1:
        x = x.contiguous()
    m = x.shape[0]
    out = torch.empty(m, dtype=torch.int64, device=x.device)
    scratch = torch.empty(64 * 64, dtype=torch.int64, device=x.device)
    for s in range(0, m, 64):
        n = min(64, m - s)
        _lib.call("mtpb_argmax", _comm_handle(comm), x[s].data_ptr(), n, v, x.stride(0), vstart,
                  out[s].data_ptr(), scratch.data_ptr(), _lib.dtype_code(x.dtype), _lib.stream_ptr(x.device))
    return out.view(*local_logits.shape[:-1], 1)


def qkv_rope(
    x: torch.Tensor,  # [B, T, H]
    w: torch.Tensor,
    bias: torch.Tensor | None,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    hq: int,
    hkv: int,
    cache_len: int,
    rope_pos: torch.Tensor | None,
    cos: torch.Tensor,
    sin: torch.Tensor,
    comm=None,
) -> torch.Tensor:
    """Fused QKV GEMV + bias + RoPE; writes K/V at slots [cache_len, cache_len + T)."""
    _lib.require_cuda(x, w, k_cache, v_cache)
    b, t, h = x.shape
    hd = k_cache.shape[-1]
    cap = k_cache.shape[2]
    q = torch.empty(b, t, hq * hd, dtype=x.dtype, device=x.device)
    xc = _c(x)
    rp = None if rope_pos is None else _c(rope_pos.to(torch.int64))
    _lib.call(
        "mtpb_qkv_rope", xc.data_ptr(), h, _c(w).data_ptr(), _lib.ptr(None if bias is None else _c(bias)),
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), b, t, hq, hkv, hd, h, cap, cache_len,
        _lib.ptr(rp), cos.data_ptr(), sin.data_ptr(), cos.shape[0], _lib.dtype_code(x.dtype), _comm_handle(comm),
        _lib.stream_ptr(x.device),
    )
    return q


def attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, hq: int, hkv: int,
              cache_len: int, comm=None) -> torch.Tensor:
    """q [B, T, hq*hd] against cache slots [0, cache_len + t] -> [B, T, hq*hd]."""
    _lib.require_cuda(q, k_cache, v_cache)
    b, t, _ = q.shape
    hd = k_cache.shape[-1]
    out = torch.empty_like(q)
    _lib.call("mtpb_attention", _c(q).data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), b, t, hq,
              hkv, hd, k_cache.shape[2], cache_len, _lib.dtype_code(q.dtype), _comm_handle(comm),
              _lib.stream_ptr(q.device))
    return out


# ---------------------------------------------------------------------- #
# beam search, and attention over a shared prefix (no counterpart in the reference)
# ---------------------------------------------------------------------- #
def _same_device(name: str, *tensors: torch.Tensor | None) -> torch.device:
    """The tensors' one CUDA device; raises when there is none or another."""
    dev = tensors[0].device
    if dev.type != "cuda":
        _lib.require_cuda(tensors[0])
    for t in tensors[1:]:
        if t is not None and t.device != dev:
            _lib.require_cuda(t)
            raise _lib.MinitpB200Error(f"{name}: tensors on {dev} and {t.device}")
    return dev


def _call_on(dev: torch.device, name: str, *args) -> None:
    """Call a C entry with ``dev`` current and its current stream as the last argument."""
    stream = torch._C._cuda_getCurrentRawStream(dev.index)
    if torch._C._cuda_getDevice() == dev.index:
        rc = getattr(_lib.load(), name)(*args, stream)
    else:
        with torch.cuda.device(dev):
            rc = getattr(_lib.load(), name)(*args, stream)
    if rc:
        _lib.check(rc)


def _beam_inputs(name: str, logits, scores, k, finished, eos_token_id, least: int = 1):
    """Checks shared by the beam selection calls -> (device, logits as rows, row stride)."""
    if logits.dim() != 3 or scores.dim() != 2 or scores.shape != logits.shape[:2]:
        raise _lib.MinitpB200Error(f"{name}: need logits [G, W, V] and scores [G, W], got {tuple(logits.shape)} and "
                                   f"{tuple(scores.shape)}")
    dev = _same_device(name, logits, scores, finished)
    if scores.dtype != torch.float32 or not scores.is_contiguous():
        raise _lib.MinitpB200Error(f"{name}: scores must be contiguous fp32")
    g, w, v = logits.shape
    if not (1 <= w <= 64 and 1 <= k <= 64 and g >= 1 and least <= v < 2**30):
        raise _lib.MinitpB200Error(f"{name}: need 1..64 beams, k in [1, 64] and a vocabulary of 1 .. 2^30 - 1")
    if finished is not None:
        if finished.dtype != torch.bool or finished.shape != scores.shape or not finished.is_contiguous():
            raise _lib.MinitpB200Error(f"{name}: finished must be contiguous bool [G, W]")
        if eos_token_id is None:
            raise _lib.MinitpB200Error(f"{name}: finished beams need eos_token_id")
    if eos_token_id is not None and not 0 <= eos_token_id < 2**32 - 1:
        raise _lib.MinitpB200Error(f"{name}: eos_token_id {eos_token_id} out of range")
    # rows of one stride are read in place; anything else is packed first
    if logits.stride(2) != 1 or (g > 1 and w > 1 and logits.stride(0) != w * logits.stride(1)):
        logits = logits.contiguous()
    ld = logits.stride(1) if w > 1 else logits.stride(0) if g > 1 else v
    if ld < v:  # an expanded dimension
        logits, ld = logits.contiguous(), v
    return dev, logits, ld


def _beam_outputs(dev, g: int, k: int, flags: bool):
    # (empty_strided takes half of empty's time, which counts in a call of 20 us)
    size, stride = (g, k), (k, 1)
    parents = torch.empty_strided(size, stride, dtype=torch.int64, device=dev)
    return (torch.empty_strided(size, stride, dtype=torch.float32, device=dev), parents, torch.empty_like(parents),
            torch.empty_strided(size, stride, dtype=torch.bool, device=dev) if flags else None)


def beam_select(logits: torch.Tensor, scores: torch.Tensor, k: int, finished: torch.Tensor | None = None,
                eos_token_id: int | None = None):
    """One beam-search step: the ``k`` best continuations of each prompt.

    ``logits [G, W, V]`` (fp32 or bf16) of W beams, running ``scores [G, W]``
    (fp32 sums of log-probabilities; -inf: an unused beam). A candidate (b, v)
    scores ``scores[b] + log_softmax(logits[b])[v]``; equal scores go to the
    lower ``b * V + v``. A beam flagged in ``finished`` (bool [G, W]) has one
    candidate, ``eos_token_id`` at its own score.

    Returns ``(scores, parents, tokens, finished)``, each ``[G, k]``, best
    first (``finished`` is None without ``eos_token_id``). Places without a
    candidate hold score -inf, parent 0 and the end token (or 0). At most 65535
    beams in all (G * W), 64 of a prompt, and 64 candidates.
    """
    dev, logits, ld = _beam_inputs("beam_select", logits, scores, k, finished, eos_token_id)
    g, w, v = logits.shape
    out, parents, tokens, done = _beam_outputs(dev, g, k, eos_token_id is not None)
    block = torch.empty_strided((beam_block_bytes(g * w, v, k),), (1,), dtype=torch.uint8, device=dev)
    _call_on(dev, "mtpb_beam_select", logits.data_ptr(), ld, g, w, v, scores.data_ptr(), _lib.ptr(finished),
             -1 if eos_token_id is None else eos_token_id, k, out.data_ptr(), parents.data_ptr(), tokens.data_ptr(),
             _lib.ptr(done), block.data_ptr(), _lib.dtype_code(logits.dtype))
    return out, parents, tokens, done


def beam_block_bytes(rows: int, v_plan: int, k: int) -> int:
    """Bytes of one shard's candidate block (``beam_candidates``)."""
    n = _lib.load().mtpb_beam_block_bytes(rows, v_plan, k)
    if n < 0:
        _lib.check(n)
    return n


def beam_candidates(local_logits: torch.Tensor, k: int, vstart: int, v_plan: int,
                    finished: torch.Tensor | None = None) -> torch.Tensor:
    """One vocabulary shard ``[G, W, V_local]`` (columns from ``vstart``; it may be empty) reduced to a
    block of candidates (uint8 [n]). ``v_plan``: the largest shard's columns, the same on every rank."""
    if local_logits.dim() != 3 or not (0 <= vstart < 2**32 and 1 <= v_plan < 2**30):
        raise _lib.MinitpB200Error(f"beam_candidates: need logits [G, W, V_local], a start below 2^32 and a plan of at "
                                   f"least one column, got {tuple(local_logits.shape)}, {vstart} and {v_plan}")
    g, w, v = local_logits.shape
    zeros = local_logits.new_empty((g, w), dtype=torch.float32)  # stands for the scores in the checks
    dev, x, ld = _beam_inputs("beam_candidates", local_logits, zeros, k, finished, 0, least=0)
    block = torch.empty(beam_block_bytes(g * w, v_plan, k), dtype=torch.uint8, device=dev)
    _call_on(dev, "mtpb_beam_candidates", x.data_ptr(), ld, g * w, v, vstart, v_plan, k, _lib.ptr(finished),
             block.data_ptr(), _lib.dtype_code(x.dtype))
    return block


def beam_pick(blocks: torch.Tensor, scores: torch.Tensor, k: int, v_plan: int, finished: torch.Tensor | None = None,
              eos_token_id: int | None = None):
    """``beam_select``'s result from the candidate blocks ``[shards, n]`` of every vocabulary shard."""
    dev = _same_device("beam_pick", blocks, scores, finished)
    if scores.dim() != 2 or not (1 <= k <= 64 and 1 <= v_plan < 2**30):
        raise _lib.MinitpB200Error(f"beam_pick: need scores [G, W] and k in [1, 64], got {tuple(scores.shape)} and {k}")
    if eos_token_id is not None and not 0 <= eos_token_id < 2**32 - 1:
        raise _lib.MinitpB200Error(f"beam_pick: eos_token_id {eos_token_id} out of range")
    g, w = scores.shape
    if blocks.dim() != 2 or blocks.dtype != torch.uint8 or not blocks.is_contiguous() or \
            blocks.shape[1] != beam_block_bytes(g * w, v_plan, k):
        raise _lib.MinitpB200Error("beam_pick: blocks must be contiguous uint8 [shards, beam_block_bytes(rows, v_plan, k)]")
    if scores.dtype != torch.float32 or not scores.is_contiguous():
        raise _lib.MinitpB200Error("beam_pick: scores must be contiguous fp32")
    if finished is not None and (finished.dtype != torch.bool or finished.shape != scores.shape
                                 or not finished.is_contiguous() or eos_token_id is None):
        raise _lib.MinitpB200Error("beam_pick: finished must be contiguous bool [G, W], with eos_token_id")
    out, parents, tokens, done = _beam_outputs(dev, g, k, eos_token_id is not None)
    _call_on(dev, "mtpb_beam_pick", blocks.data_ptr(), blocks.shape[0], g, w, v_plan, k, scores.data_ptr(),
             _lib.ptr(finished), -1 if eos_token_id is None else eos_token_id, k, out.data_ptr(), parents.data_ptr(),
             tokens.data_ptr(), _lib.ptr(done))
    return out, parents, tokens, done


def _length_arg(name: str, lengths, count: int, cap: int, dev):
    """(device pointer or None, host value) of a per-row length argument."""
    if isinstance(lengths, int):
        if not 0 <= lengths <= cap:
            raise _lib.MinitpB200Error(f"{name}: length {lengths} outside the cache of {cap} positions")
        return None, lengths
    if not isinstance(lengths, torch.Tensor) or lengths.dtype != torch.int32 or lengths.shape != (count,) or not lengths.is_contiguous() or \
            lengths.device != dev:
        raise _lib.MinitpB200Error(f"{name}: lengths must be an int or contiguous int32 [{count}] on {dev}")
    return lengths.data_ptr(), 0


# what a reordering asks of each of a model's caches (a loop over the 48 of the 0.5B shape costs three times this)
_SHAPE, _DTYPE = operator.attrgetter("shape"), operator.attrgetter("dtype")


def reorder_cache_(k_caches, v_caches, parents: torch.Tensor, lengths) -> None:
    """In place, in every layer: row ``g * W + w`` becomes row ``g * W + parents[g, w]``.

    ``k_caches`` / ``v_caches``: lists of ``[G * W, hkv, cap, hd]`` caches;
    ``parents`` int64 ``[G, W]``. The first ``lengths`` positions of the source
    row are copied (an int, or int32 ``[G * W]`` by source row); later ones stay
    as they were. A parent outside [0, W) leaves its row alone. No two caches may
    share memory. W is at most 64, G * hkv at most 65535.
    """
    name = "reorder_cache_"
    if parents.dim() != 2 or parents.dtype != torch.int64 or not parents.is_contiguous():
        raise _lib.MinitpB200Error(f"{name}: parents must be contiguous int64 [G, W]")
    caches = [*k_caches, *v_caches]
    n = len(k_caches)
    if n == 0 or len(v_caches) != n:
        raise _lib.MinitpB200Error(f"{name}: need as many K as V caches")
    first = caches[0]
    dev = _same_device(name, parents, first)
    shape, dtype = first.shape, first.dtype
    g, w = parents.shape
    if first.dim() != 4 or shape[0] != g * w:
        raise _lib.MinitpB200Error(f"{name}: caches must be [{g * w}, hkv, cap, hd], got {tuple(shape)}")
    if set(map(_SHAPE, caches)) != {shape} or set(map(_DTYPE, caches)) != {dtype} or \
            set(map(torch.Tensor.get_device, caches)) != {dev.index} or not all(map(torch.Tensor.is_contiguous, caches)):
        raise _lib.MinitpB200Error(f"{name}: caches must be contiguous, of one shape, dtype and device")
    lens, length = _length_arg(name, lengths, g * w, shape[2], dev)
    ptrs = array.array("Q", map(torch.Tensor.data_ptr, caches))
    at, _ = ptrs.buffer_info()
    _call_on(dev, "mtpb_kv_reorder", at, at + 8 * n, n, parents.data_ptr(), lens, length, g, w,
             shape[1], shape[2], shape[3], _lib.dtype_code(dtype))


def shared_prefix_attention(q: torch.Tensor, k_prefix: torch.Tensor, v_prefix: torch.Tensor, prefix_lens,
                            k_cache: torch.Tensor, v_cache: torch.Tensor, cache_lens, hq: int,
                            hkv: int) -> torch.Tensor:
    """Grouped-query attention of rows that share a prefix -> ``[N, T, hq * hd]``.

    ``q [N, T, hq * hd]``; prefix caches ``[G, hkv, cap_p, hd]``, one for every
    ``N / G`` consecutive rows; own caches ``[N, hkv, cap, hd]``. Token t of row
    n sees positions ``[0, prefix_lens[g])`` of the prefix and
    ``[0, cache_lens[n] - (T - 1 - t))`` of its own cache (which holds the T
    tokens already); one that sees nothing gets 0. Lengths are ints within their
    cache, or int32 tensors ``[G]`` / ``[N]``, clamped to it.
    """
    name = "shared_prefix_attention"
    dev = _same_device(name, q, k_prefix, v_prefix, k_cache, v_cache)
    if q.dim() != 3 or k_prefix.dim() != 4 or k_cache.dim() != 4:
        raise _lib.MinitpB200Error(f"{name}: need q [N, T, hq*hd] and caches [rows, hkv, cap, hd]")
    n, t, _ = q.shape
    g, _, cap_p, hd = k_prefix.shape
    cap = k_cache.shape[2]
    if g < 1 or n < 1 or t < 1 or n % g or hq < 1 or hkv < 1 or hq % hkv:
        raise _lib.MinitpB200Error(f"{name}: {n} rows of {t} tokens in {g} groups, {hq} heads over {hkv}")
    if q.shape[2] != hq * hd or k_prefix.shape != (g, hkv, cap_p, hd) or v_prefix.shape != k_prefix.shape or \
            k_cache.shape != (n, hkv, cap, hd) or v_cache.shape != k_cache.shape:
        raise _lib.MinitpB200Error(f"{name}: shapes {tuple(q.shape)}, {tuple(k_prefix.shape)}, {tuple(k_cache.shape)} "
                                   "do not fit together")
    for c in (k_prefix, v_prefix, k_cache, v_cache):
        if c.dtype != q.dtype or not c.is_contiguous():
            raise _lib.MinitpB200Error(f"{name}: caches must be contiguous and of q's dtype")
    q = _c(q)
    plen, plen_all = _length_arg(name, prefix_lens, g, cap_p, dev)
    clen, clen_all = _length_arg(name, cache_lens, n, cap, dev)
    code = _lib.dtype_code(q.dtype)
    need = _lib.load().mtpb_shared_attention_workspace(g, n // g, t, hq, hkv, hd, cap_p, cap, code)
    if need < 0:
        _lib.check(need)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    out = torch.empty_like(q)
    _call_on(dev, "mtpb_shared_attention", q.data_ptr(), k_prefix.data_ptr(), v_prefix.data_ptr(), plen, plen_all,
             k_cache.data_ptr(), v_cache.data_ptr(), clen, clen_all, out.data_ptr(), g, n // g, t, hq, hkv, hd, cap_p,
             cap, code, _lib.ptr(ws), need)
    return out
