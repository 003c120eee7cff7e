"""Packed prompt attention and token log-probabilities where their schedules and masks have an edge."""

import ctypes
import math

import pytest
import torch

from tests import scoring_ref
from tests.test_gpu_scoring import DT, _close, _cuda_starts, _gen, _parts, _starts

pytestmark = pytest.mark.gpu


def _status_is_clean(lib):
    s = ctypes.c_uint32(7)
    assert lib.mtpb_scoring_status(ctypes.byref(s)) == 0 and s.value == 0


# ------------------------------------------------------------------ log-probabilities
def _check_some(got, x, t, top, step=13):
    """Every `step`-th row, and the last, against the definition."""
    at = torch.tensor(sorted({*range(0, x.shape[0], step), x.shape[0] - 1}), device=x.device)
    scoring_ref.check_logprobs([None if g is None else g[at] for g in got], x[at], t[at], top)


@pytest.mark.parametrize("dtype,rows,v,pad", [("bf16", 8192, 8195, 0), ("bf16", 2730, 49153, 0), ("bf16", 2047, 65537, 0),
                                              ("fp32", 4096, 4097, 0), ("bf16", 4096, 16390, 1), ("bf16", 3000, 8200, 1),
                                              ("fp32", 620, 49155, 0), ("bf16", 1500, 8192, 3)])
@pytest.mark.parametrize("top", [0, 5, 64])
def test_rows_that_end_just_past_a_tile(lib, dtype, rows, v, pad, top):
    """Rows whose last tile holds no whole vector, or none at some starts in memory; several rows to a CTA."""
    from minitp_b200 import ops

    r = torch.Generator(device="cuda").manual_seed(rows + v)
    wide = torch.empty(rows, v + pad, dtype=DT[dtype], device="cuda")
    wide.normal_(0.0, 3.0, generator=r)
    x = wide[:, pad:]
    t = torch.randint(0, v, (rows,), generator=r, device="cuda")
    t[::3] = v - 1
    x[::4, -1] = 20.0  # the best, outside the whole vectors
    _check_some(ops.token_logprobs(x, t, top), x, t, top)
    _status_is_clean(lib)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("top", [0, 5, 64])
def test_shards_of_fewer_tiles_than_planned(lib, dtype, top):
    """Shards of no, few and most of the planned columns, with many rows to a CTA."""
    from minitp_b200 import ops

    rows, plan, cuts = 4096, 20000, [0, 9000, 9000, 17200, 17203]
    r = torch.Generator(device="cuda").manual_seed(top)
    x = torch.empty(rows, cuts[-1], dtype=DT[dtype], device="cuda").normal_(0.0, 3.0, generator=r)
    t = torch.randint(0, cuts[-1], (rows,), generator=r, device="cuda")
    blocks = [ops.logprobs_block(x[:, a:b], t, top, a, plan) for a, b in zip(cuts, cuts[1:])]
    _check_some(ops.logprobs_join(torch.stack(blocks), t, (rows,), top, plan, DT[dtype]), x, t, top, 41)
    _status_is_clean(lib)


# ------------------------------------------------------------------ attention
# (query heads, KV heads, head dim, prompts) on the tensor cores; more than 256 x 148 (token, head) rows take
# items of 256 rows, fewer items of 128
LARGE = [(14, 2, 64, [600, 1, 0, 700, 300, 129, 850, 400]), (16, 2, 128, [513, 900, 1, 256, 128, 0, 640]),
         (28, 4, 128, [301, 700, 420])]
SMALL = [(4, 2, 64, [300, 600]), (4, 2, 128, [600, 300])]


def _case(hq, hkv, hd, lengths, seed, large, at=0, behind=0):
    starts = _starts(lengths, at=at)
    total = starts[-1] + behind
    assert (total * hq > 256 * 148) == large
    return starts, *(t.clone() for t in _parts(_gen(seed), total, hq, hkv, hd, "bf16"))


@pytest.mark.parametrize("large,hq,hkv,hd,lengths", [(True, *c) for c in LARGE] + [(False, *c) for c in SMALL])
def test_rows_without_a_score_above_minus_infinity(lib, large, hq, hkv, hd, lengths):
    """Tokens whose scores are all -inf get 0, however many keys they see; those with one finite score that key's V."""
    from minitp_b200 import ops

    starts, q, k, v = _case(hq, hkv, hd, lengths, 60 + hd, large)
    per = hq // hkv
    q[..., 0] = 1.0
    whole = lengths.index(max(lengths))  # a prompt whose keys are all -inf for the first KV head
    a, b = starts[whole], starts[whole + 1]
    k[a:b, 0, 0] = -math.inf
    k[a:b - 40, 1, 0] = -math.inf  # for the second one up to the last 40
    k[starts[0]:starts[0] + 250, 0, 0] = -math.inf  # another prompt's first 250
    got = ops.prompt_attention(q, k, v, _cuda_starts(starts))
    assert not got[a:b, :per].any() and not got[a:b - 40, per:2 * per].any()
    _close(got, *scoring_ref.attend(q, k, v, starts))


@pytest.mark.parametrize("hq,hkv,hd,lengths", LARGE)
def test_large_items_nan_and_infinities(lib, hq, hkv, hd, lengths):
    """Of K and V, in the middle of prompts, at tiles' edges and at their last tokens, for one KV head each."""
    from minitp_b200 import ops

    starts, q, k, v = _case(hq, hkv, hd, lengths, 70 + hd, True)
    per, last = hq // hkv, hkv - 1
    ends = [b for a, b in zip(starts, starts[1:]) if b > a]
    v[100, 0, 3] = math.nan
    v[127, 0, 5] = math.inf
    v[128, last, 7] = -math.inf
    for i, b in enumerate(ends):  # seen by the last token alone
        v[b - 1, i % hkv, 8 + i] = (math.nan, math.inf, -math.inf)[i % 3]
    a = starts[-2]
    k[a + 290, 0, 2] = math.nan  # later tokens' scores
    got = ops.prompt_attention(q, k, v, _cuda_starts(starts))
    want, tol = scoring_ref.attend(q, k, v, starts)
    want[a + 290:starts[-1], :per] = math.nan
    _close(got, want, tol)


@pytest.mark.parametrize("hq,hkv,hd,lengths", LARGE)
def test_large_items_large_scores(lib, hq, hkv, hd, lengths):
    """Scores of some thousands that grow along the tokens (the running maximum moves at every tile) or fall."""
    from minitp_b200 import ops

    starts, q, k, v = _case(hq, hkv, hd, lengths, 80 + hd, True)
    q[..., 0] = 40.0
    for sign in (1, -1):
        k[..., 0] = (sign * torch.arange(starts[-1]) * 0.5).to(k.dtype).cuda()[:, None]
        _close(ops.prompt_attention(q, k, v, _cuda_starts(starts)), *scoring_ref.attend(q, k, v, starts))


@pytest.mark.parametrize("hq,hkv,hd,lengths", LARGE)
def test_large_items_strides(lib, hq, hkv, hd, lengths):
    """Heads before tokens, padded rows beside NaN, an unaligned view and strided dims: one result."""
    from minitp_b200 import ops

    starts, q, k, v = _case(hq, hkv, hd, lengths, 90 + hd, True)
    st, n = _cuda_starts(starts), starts[-1]
    want = ops.prompt_attention(q, k, v, st)
    _close(want, *scoring_ref.attend(q, k, v, starts))

    def padded(t):
        w = torch.full((n + 3, t.shape[1] + 2, hd + 16), math.nan, dtype=t.dtype, device="cuda")
        w[1:n + 1, 1:-1, 16:] = t
        return w[1:n + 1, 1:-1, 16:]

    def unaligned(t):
        w = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        w[1:] = t.reshape(-1)
        return w[1:].view(t.shape)

    for f in (lambda t: t.transpose(0, 1).contiguous().transpose(0, 1), padded, unaligned,
              lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)):
        assert torch.equal(ops.prompt_attention(f(q), f(k), f(v), st), want)


@pytest.mark.parametrize("hq,hkv,hd,lengths", LARGE)
def test_large_items_tokens_of_no_prompt_and_pieces(lib, hq, hkv, hd, lengths):
    """NaN before, behind and (by the pieces) around what is asked for; tokens of no prompt become 0."""
    from minitp_b200 import ops

    starts, q, k, v = _case(hq, hkv, hd, lengths, 100 + hd, True, at=130, behind=77)
    for t in (q, k, v):
        t[:130] = math.nan
        t[starts[-1]:] = math.nan
    want, tol = scoring_ref.attend(q, k, v, starts)
    got = ops.prompt_attention(q, k, v, _cuda_starts(starts))
    assert not got[:130].any() and not got[starts[-1]:].any()
    _close(got, want, tol)
    total = q.shape[0]
    a, b = 3, total - 5
    assert (b - a) * hq > 256 * 148
    _close(ops.prompt_attention(q[a:b], k, v, _cuda_starts(starts), first=a), want[a:b], tol[a:b])


@pytest.mark.parametrize("hq,hkv,hd,lengths", LARGE)
def test_large_items_starts_out_of_range(lib, hq, hkv, hd, lengths):
    from minitp_b200 import ops

    starts, q, k, v = _case(hq, hkv, hd, lengths, 110 + hd, True)
    total = starts[-1]
    for given, meant in [([-5, 700, total + 900], [0, 700, total]), ([500, 30, 1200, total], [500, 500, 1200, total]),
                         ([total + 3, total + 9], [total, total])]:
        got = ops.prompt_attention(q, k, v, _cuda_starts(given))
        want, tol = scoring_ref.attend(q[:1500], k, v, meant)
        _close(got[:1500], want, tol)
        assert bool(torch.isfinite(got).all())


@pytest.mark.parametrize("hq,hkv,hd,lengths", LARGE)
def test_large_items_captured_and_on_another_stream(lib, hq, hkv, hd, lengths):
    """A captured call replays on new contents and new starts; another stream's call gives the same."""
    from minitp_b200 import ops

    starts, q, k, v = _case(hq, hkv, hd, lengths, 120 + hd, True)
    n, st = starts[-1], _cuda_starts(starts)
    ops.prompt_attention(q, k, v, st)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.prompt_attention(q, k, v, st)
    side = torch.cuda.Stream()
    other_starts = [starts[0] + 1, *sorted(s // 2 for s in starts[1:-1]), n - 1]
    for seed, new in [(121, starts), (122, sorted(other_starts))]:
        nq, nk, nv = _parts(_gen(seed), n, hq, hkv, hd, "bf16")
        q.copy_(nq), k.copy_(nk), v.copy_(nv), st.copy_(_cuda_starts(new))
        g.replay()
        _close(out, *scoring_ref.attend(nq, nk, nv, new))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = ops.prompt_attention(q, k, v, st)
        side.synchronize()
        assert torch.equal(other, out)

@pytest.mark.parametrize("dtype,hq,hkv,hd", [("fp32", 4, 2, 16), ("bf16", 6, 3, 32), ("fp32", 7, 1, 128), ("bf16", 14, 2, 64),
                                             ("bf16", 4, 1, 128)])
def test_prompts_around_the_number_that_is_put_in_order(lib, dtype, hq, hkv, hd):
    """31 to 33 and 63 to 65 prompts, and more; empty ones among them, a long one last, whole calls and pieces."""
    from minitp_b200 import ops

    for count in (31, 32, 33, 63, 64, 65, 129, 300):
        r = _gen(count)
        lengths = torch.randint(0, 9, (count,), generator=r).tolist()
        lengths[count // 3] = 0
        lengths[count - 1] = 150
        starts = _starts(lengths, at=2)
        q, k, v = _parts(r, starts[-1] + 3, hq, hkv, hd, dtype)
        want, tol = scoring_ref.attend(q, k, v, starts)
        _close(ops.prompt_attention(q, k, v, _cuda_starts(starts)), want, tol)
        a, b = starts[count // 4] + 1, starts[-1] - 20
        _close(ops.prompt_attention(q[a:b], k, v, _cuda_starts(starts), first=a), want[a:b], tol[a:b])


@pytest.mark.parametrize("dtype,hq,hkv,hd", [("fp32", 4, 2, 16), ("bf16", 4, 2, 64)])
def test_as_many_prompts_as_a_scoring_forward_takes(lib, dtype, hq, hkv, hd):
    """2^16 prompts of a few tokens: a token sees its own prompt, by the plain sums over up to four keys."""
    from minitp_b200 import ops

    count = 1 << 16
    g = torch.Generator(device="cuda").manual_seed(1)
    lengths = torch.randint(0, 5, (count,), generator=g, device="cuda")
    starts = torch.cat([lengths.new_zeros(1), lengths.cumsum(0)]).int()
    n = int(starts[-1])
    q, k, v = (torch.randn(n, h, hd, generator=g, device="cuda").to(DT[dtype]) for h in (hq, hkv, hkv))
    got = ops.prompt_attention(q, k, v, starts)
    tok = torch.arange(n, device="cuda")
    first = starts.long().repeat_interleave(torch.cat([lengths, lengths.new_zeros(1)]))
    per = hq // hkv
    kd, vd = (x.double().repeat_interleave(per, 1) for x in (k, v))
    back = tok[:, None] - torch.arange(4, device="cuda")  # a token and the three before it
    seen = (back >= first[:, None])[:, None]
    back = back.clamp(min=0)
    s = (q.double()[:, :, None] * kd[back].transpose(1, 2)).sum(-1) / math.sqrt(hd)
    p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
    want = (p[..., None] * vd[back].transpose(1, 2)).sum(2)
    # (scoring_ref.attend's tolerance with |q k| <= 6 sqrt(hd) |q|, |v| <= 6 for these values: 4 keys)
    half = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -24
    mag = (q.double().abs()[:, :, None] * kd.abs()[back].transpose(1, 2)).sum(-1).amax(-1, keepdim=True) / math.sqrt(hd)
    rel = 2 * (hd + 4) * 2.0 ** -24 * mag + 68 * 2.0 ** -24 + (2.0 ** -14 if dtype == "bf16" else 0.0)
    tol = rel * vd[back].abs().amax(dim=(1, 3))[..., None] + 1.01 * half * want.abs()
    if dtype == "bf16":
        tol = tol + 1.01 * half * (p[..., None] * vd[back].abs().transpose(1, 2)).sum(2)
    assert bool(((got.double() - want).abs() <= tol).all())
    _status_is_clean(lib)


@pytest.mark.parametrize("dtype,hq,hkv,hd", [("fp32", 4, 2, 16), ("fp32", 28, 4, 128), ("bf16", 14, 2, 64)])
def test_few_tokens_of_many_are_in_a_prompt(lib, dtype, hq, hkv, hd):
    """Tokens of no prompt in the thousands, before and behind few or many prompts, and no prompt at all, become 0."""
    from minitp_b200 import ops

    for total, starts in [(1, [0]), (3, [3]), (5000, [2500, 2520]), (5000, [4999]), (3000, list(range(1000, 1100)))]:
        q, k, v = _parts(_gen(total), total, hq, hkv, hd, dtype)
        for t in (q, k, v):
            t[:starts[0]] = math.nan
            t[starts[-1]:] = math.nan
        want, tol = scoring_ref.attend(q, k, v, starts)
        torch.empty(total, hq, hd, dtype=DT[dtype], device="cuda").fill_(math.nan)  # (what the output's memory may hold)
        _close(ops.prompt_attention(q, k, v, _cuda_starts(starts)), want, tol)


# ------------------------------------------------------------------ errors that only the device knows of
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("top", [0, 3, 64])
def test_rows_of_lost_parts_are_nan(lib, dtype, top):
    """Statistics that say that a part's logits never came make their row NaN, alternatives too, and no other row."""
    from minitp_b200 import ops

    rows, v = 40, 60000
    x = torch.randn(rows, v, generator=_gen(top)).to(DT[dtype]).cuda()
    t = torch.arange(rows, device="cuda") * 7
    blocks = torch.stack([ops.logprobs_block(x[:, :30000], t, top, 0, 30000), ops.logprobs_block(x[:, 30000:], t, top, 30000, 30000)])
    want = ops.logprobs_join(blocks, t, (rows,), top, 30000, DT[dtype])
    # a row has a part at least; its statistics are {max, sum, mean, target}, at the block's start
    parts = (blocks.shape[1] // rows) // (16 + 8 * top)
    for row in (0, 17, rows - 1):
        at = row * parts * 16 + 4
        blocks[row % 2, at:at + 4] = torch.tensor([255, 255, 255, 127], dtype=torch.uint8)  # the sum: NaN
    got = ops.logprobs_join(blocks, t, (rows,), top, 30000, DT[dtype])
    lost = torch.zeros(rows, dtype=torch.bool, device="cuda")
    lost[[0, 17, rows - 1]] = True
    for g, w in zip(got[:3], want[:3]):
        if g is not None:
            assert bool(g[lost].isnan().all()) and torch.equal(g[~lost], w[~lost])
    if top:
        assert torch.equal(got[3][~lost], want[3][~lost])


def test_a_wait_that_ran_out_raises(lib, monkeypatch):
    """`raise_on_scoring_error` by a status that a stand-in of the library call hands back, and by the real one."""
    from minitp_b200 import _lib, ops

    ops.raise_on_scoring_error("cuda")
    call = _lib.call

    def fake(name, *args):
        if name == "mtpb_scoring_status":
            args[0]._obj.value = _lib.STATUS_TIMEOUT
            return
        call(name, *args)

    monkeypatch.setattr(_lib, "call", fake)
    with pytest.raises(_lib.MinitpB200Error, match="ran out"):
        ops.raise_on_scoring_error("cuda")


def _tiny_model():
    from minitp_b200 import config as mcfg
    from minitp_b200.distributed.context import context_for
    from minitp_b200.weight_loader import load_synthetic_tp

    cfg = mcfg.baseline_tiny()
    return load_synthetic_tp(cfg, context_for(1, "cuda"), dtype=torch.float32, device=torch.device("cuda")), cfg


def test_scores_whose_forward_reported_an_error_are_not_returned(lib, monkeypatch):
    """A forward that flags its communicator makes `score_prompts` raise; a word set before does not."""
    from minitp_b200 import _lib, ops
    from minitp_b200.scoring import score_prompts

    model, cfg = _tiny_model()
    comm = model.ctx.comm()
    prompts = [[1, 2, 3], [4, 5]]
    want = score_prompts(model, prompts)
    real = model.forward_packed

    def behind_the_table(ids, starts):
        return real(ids, starts, torch.full_like(ids, cfg.max_position_embeddings + 5))

    try:
        monkeypatch.setattr(model, "forward_packed", behind_the_table)
        with pytest.raises(_lib.MinitpB200Error, match="position"):
            score_prompts(model, prompts)
        monkeypatch.undo()
        again = score_prompts(model, prompts)  # (the word still holds what the call before reported)
        assert all(torch.equal(a.logprobs, w.logprobs) for a, w in zip(again, want))
    finally:
        comm.clear_status()
    status = _lib.call

    def ran_out(name, *args):
        if name == "mtpb_scoring_status":
            args[0]._obj.value = _lib.STATUS_TIMEOUT
            return
        status(name, *args)

    monkeypatch.setattr(_lib, "call", ran_out)
    with pytest.raises(_lib.MinitpB200Error, match="ran out"):
        score_prompts(model, prompts)


def test_ids_outside_the_vocabulary_are_refused_on_either_device(lib):
    from minitp_b200.scoring import score_prompts

    model, cfg = _tiny_model()
    for wrong in (-1, cfg.vocab_size, 2 ** 40, -2 ** 40):
        for device in ("cpu", "cuda"):
            with pytest.raises(ValueError, match="vocabulary"):
                score_prompts(model, [[1, 2], torch.tensor([3, wrong], device=device), torch.tensor([5], device="cuda")])
    assert model.ctx.comm().status() == 0
    last = torch.tensor([0, cfg.vocab_size - 1])
    for ids in (last, last.cuda(), last.to(torch.int16 if cfg.vocab_size < 2 ** 15 else torch.int32).cuda(), last.tolist()):
        assert bool(torch.isfinite(score_prompts(model, [ids])[0].logprobs).all())


def test_sizes_past_the_c_types_are_refused(lib):
    """Sizes whose lower 32 bits look fine are refused, not cut to those (expanded tensors: no memory behind them)."""
    from minitp_b200 import _lib, ops

    far = 2 ** 32
    q, k = torch.zeros(5, 2, 64, device="cuda"), torch.zeros(5, 1, 64, device="cuda")
    st = _cuda_starts([0, 5])
    wide = torch.zeros(1, device="cuda").expand(5, 1, far + 64)
    for args, match in [((q, k[:1].expand(far + 5, 1, 64), k[:1].expand(far + 5, 1, 64), st), "rows"),
                        ((q[:, :1].expand(5, far + 2, 64), k, k, st), "heads"), ((wide, wide, wide, st), "head_dim"),
                        ((q, k, k, torch.zeros(2 ** 20 + 2, dtype=torch.int32, device="cuda")), "prompts")]:
        with pytest.raises(_lib.MinitpB200Error, match=match):
            ops.prompt_attention(*args)
    x, t = torch.zeros(1, 10, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    for rows in (far + 8, 2 ** 24 + 1):
        for call in (lambda: ops.token_logprobs(x.expand(rows, 10), t.expand(rows), 2),
                     lambda: ops.logprobs_block(x.expand(rows, 10), None, 2, 0, 10),
                     lambda: ops.logprobs_join(torch.zeros(1, 16, dtype=torch.uint8, device="cuda"), None, (rows,), 2, 10,
                                               torch.float32)):
            with pytest.raises(_lib.MinitpB200Error, match="rows"):
                call()
    with pytest.raises(_lib.MinitpB200Error, match="shards"):
        ops.logprobs_join(torch.zeros(65, 16, dtype=torch.uint8, device="cuda"), None, (1,), 0, 10, torch.float32)


@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
def test_a_packed_forward_that_is_refused_launches_nothing(lib):
    """Limits of the attention are looked at before the first kernel: a capture of the refused call holds no node."""
    from cuda.bindings import runtime

    from minitp_b200 import _lib

    model, cfg = _tiny_model()
    ids = torch.arange(8, device="cuda")
    few, many = _cuda_starts([0, 8]), torch.zeros(2 ** 20 + 2, dtype=torch.int32, device="cuda")
    want = model.forward_packed(ids, few, ids)

    def nodes(starts, refused):
        g = torch.cuda.CUDAGraph(keep_graph=True)
        with torch.cuda.graph(g):
            if refused:
                with pytest.raises(_lib.MinitpB200Error, match="prompts"):
                    model.forward_packed(ids, starts, ids)
            else:
                model.forward_packed(ids, starts, ids)
        err, _, count = runtime.cudaGraphGetNodes(g.raw_cuda_graph(), 0)
        assert int(err) == 0
        return count

    assert nodes(few, False) > 0
    assert nodes(many, True) == 0
    assert torch.equal(model.forward_packed(ids, few, ids), want)
    assert model.ctx.comm().status() == 0


# ------------------------------------------------------------------ the largest sizes that are taken
@pytest.mark.parametrize("dtype,hd", [("fp32", 16), ("bf16", 64)])
def test_as_many_prompts_as_are_taken(lib, dtype, hd):
    """2^20 prompts of up to three tokens: first tokens return their V, last ones the sums over their prompt."""
    from minitp_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(2)
    lengths = torch.randint(0, 4, (1 << 20,), generator=g, device="cuda")
    starts = torch.cat([lengths.new_zeros(1), lengths.cumsum(0)]).int()
    q, k, v = (torch.randn(int(starts[-1]), h, hd, generator=g, device="cuda").to(DT[dtype]) for h in (4, 2, 2))
    got = ops.prompt_attention(q, k, v, starts)
    first = starts[:-1][lengths > 0].long()
    assert torch.equal(got[first], v[first].repeat_interleave(2, 1))
    pick = first[lengths[lengths > 0] == 3][::97]
    rows = torch.stack([pick, pick + 1, pick + 2], 1).reshape(-1)
    small = list(range(0, rows.numel() + 1, 3))
    _close(got[rows], *scoring_ref.attend(q[rows], k[rows], v[rows], small))
    _status_is_clean(lib)


def test_as_many_rows_as_are_taken(lib):
    from minitp_b200 import ops

    rows, v = 1 << 24, 17
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(rows, v, generator=g, device="cuda").bfloat16()
    t = torch.randint(0, v, (rows,), generator=g, device="cuda")
    got = ops.token_logprobs(x, t, 2)
    _check_some(got, x, t, 2, 9973)
    # all rows in fp32: off by a few of its half steps of values below 16, on either side
    assert float((got[0] - torch.log_softmax(x.float(), -1).gather(1, t[:, None])[:, 0]).abs().max()) <= 40 * 2.0 ** -24 * 16


def test_a_vocabulary_as_large_as_is_taken(lib):
    from minitp_b200 import ops

    v = (1 << 30) - 1
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.empty(1, v, dtype=torch.bfloat16, device="cuda").normal_(0.0, 2.0, generator=g)
    x[0, v - 2:] = 30.0
    x[0, 0] = 29.0
    lp, entropy, best, ids = ops.token_logprobs(x, torch.tensor([v - 1], device="cuda"), 3)
    total = mean = 0.0
    for i in range(0, v, 1 << 26):
        d = x[0, i:i + (1 << 26)].double() - 30.0
        e = d.exp()
        total += float(e.sum())
        mean += float((e * d).sum())
    logs = math.log(total)
    # a lane adds 2^30 / (444 x 256) values: scoring_ref.check_logprobs' tolerance at that depth
    off = (v / (444 * 256) + 40) * 2.0 ** -24
    assert ids.tolist() == [[v - 2, v - 1, 0]]
    assert abs(float(lp) + logs) <= off * (1 + logs) and abs(float(best[0, 2]) + 1 + logs) <= off * (2 + logs)
    assert abs(float(entropy) - (logs - mean / total)) <= off * (2 + logs)
    _status_is_clean(lib)
