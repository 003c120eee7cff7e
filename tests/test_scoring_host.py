"""Refusals of the prompt-attention and log-probability calls (host checks; no GPU, no launch)."""

import pytest
import torch

from minitp_b200 import _lib, ops

P = 1 << 20  # a 16-byte aligned stand-in for a device address; every call below is refused before it is used


def _refused(lib, name, args, match):
    assert getattr(lib, name)(*args) == _lib.ERR_INVALID
    assert match in lib.mtpb_last_error().decode()


def test_attention_refusals(lib):
    ok = dict(q=P, qt=14 * 64, qh=64, k=P, kt=128, kh=64, v=P, vt=128, vh=64, out=P, starts=P, S=2, first=0, n=10, total=10,
              hq=14, hkv=2, hd=64, dtype=_lib.MTPB_BF16, st=None)
    for change, match in [(dict(q=None), "null"), (dict(starts=None), "null"), (dict(out=None), "null"),
                          (dict(hkv=4), "multiple"), (dict(hkv=0), "size"), (dict(hd=80), "head_dim"), (dict(dtype=5), "dtype"),
                          (dict(first=1), "outside"), (dict(first=-1), "outside"), (dict(n=11), "outside"),
                          (dict(n=-1), "size"), (dict(S=-1), "size"), (dict(S=1 << 21), "prompts"), (dict(q=P + 2), "aligned"),
                          (dict(qt=14 * 64 + 4), "strides"), (dict(kh=32), "strides"), (dict(vt=0), "strides"),
                          (dict(vh=-64), "strides"), (dict(n=1, total=1 << 25), "rows"),
                          (dict(n=1, total=1, hq=1 << 17, hkv=1), "heads")]:
        _refused(lib, "mtpb_prompt_attention", list((ok | change).values()), match)
    assert lib.mtpb_prompt_attention(*(ok | dict(n=0)).values()) == 0  # nothing to do


def test_logprob_refusals(lib):
    ok = dict(logits=P, ld=100, rows=8, V=100, targets=P, k=4, lp=P, ent=P, tops=P, ids=P, block=P, dtype=_lib.MTPB_F32,
              st=None)
    for change, match in [(dict(logits=None), "null"), (dict(ent=None), "null"), (dict(lp=None), "null"),
                          (dict(tops=None), "null"), (dict(ids=None), "null"), (dict(block=None), "null"),
                          (dict(k=65), "alternatives"), (dict(k=-1), "alternatives"), (dict(rows=0), "rows"),
                          (dict(rows=(1 << 24) + 1), "rows"), (dict(V=0), "vocabulary"), (dict(V=1 << 30), "vocabulary"),
                          (dict(ld=99), "ld"), (dict(dtype=7), "dtype"), (dict(block=P + 8), "aligned")]:
        _refused(lib, "mtpb_token_logprobs", list((ok | change).values()), match)
    assert lib.mtpb_logprobs_block_bytes(8, 151936, 65, 1) < 0
    assert lib.mtpb_logprobs_block_bytes(0, 151936, 4, 1) < 0
    assert lib.mtpb_logprobs_block_bytes(8, 1 << 30, 4, 0) < 0
    assert 0 < lib.mtpb_logprobs_block_bytes(8, 151936, 0, 1) < lib.mtpb_logprobs_block_bytes(8, 151936, 64, 1)
    assert lib.mtpb_logprobs_block_bytes(8, 151936, 4, 3) < 0


def test_block_and_join_refusals(lib):
    ok = dict(logits=P, ld=50, rows=8, v=50, vstart=0, plan=60, targets=None, k=4, block=P, dtype=_lib.MTPB_BF16, st=None)
    for change, match in [(dict(v=61), "V_plan"), (dict(v=-1), "V_plan"), (dict(vstart=-1), "range"),
                          (dict(vstart=2 ** 32), "range"), (dict(block=None), "null"), (dict(rows=0), "rows")]:
        _refused(lib, "mtpb_logprobs_block", list((ok | change).values()), match)
    ok = dict(blocks=P, parts=2, rows=8, plan=60, kb=4, targets=P, k=4, lp=P, ent=P, tops=P, ids=P, dtype=0, st=None)
    for change, match in [(dict(parts=0), "shards"), (dict(parts=65), "shards"), (dict(k=5), "alternatives"),
                          (dict(blocks=None), "aligned"), (dict(lp=None), "null"), (dict(kb=65), "alternatives"),
                          (dict(ent=None), "null"), (dict(dtype=2), "dtype")]:
        _refused(lib, "mtpb_logprobs_join", list((ok | change).values()), match)


def test_cpu_tensors_are_refused(lib):
    x = torch.zeros(3, 2, 16)
    with pytest.raises(_lib.MinitpB200Error, match="CUDA"):
        ops.prompt_attention(x, x, x, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(_lib.MinitpB200Error, match="CUDA"):
        ops.token_logprobs(torch.zeros(2, 10))
    with pytest.raises(_lib.MinitpB200Error, match="CUDA"):
        ops.logprobs_block(torch.zeros(2, 10), None, 2, 0, 10)
    with pytest.raises(_lib.MinitpB200Error, match="CUDA"):
        ops.logprobs_join(torch.zeros(2, 10, dtype=torch.uint8), None, (2,), 2, 10, torch.float32)


def _cpu_block(local_logits, targets, top, vstart, v_plan):
    """A stand-in for a shard's block: its sum of exponentials, its entropy's sum, the targets' logits and its best."""
    n, v = local_logits.shape
    x = torch.full((n, v_plan + top), -torch.inf, dtype=torch.float64)
    x[:, :v] = local_logits.double()
    e = x.exp()
    mine = (targets >= vstart) & (targets < vstart + v)
    xt = torch.where(mine, x.gather(1, (targets - vstart).clamp(0, v_plan - 1)[:, None])[:, 0], torch.nan)
    val, at = x.sort(dim=-1, descending=True, stable=True)
    cols = [e.sum(-1, keepdim=True), torch.where(e > 0, e * x, 0.0).sum(-1, keepdim=True), xt[:, None], val[:, :top],
            (at[:, :top] + vstart).double()]
    return torch.cat(cols, -1).reshape(-1).view(torch.uint8)


def _cpu_join(blocks, targets, shape, top, v_plan, dtype):
    rows = blocks.contiguous().view(torch.float64).view(blocks.shape[0], *shape, 3 + 2 * top)
    total = rows[..., 0].sum(0)
    xt = torch.nan_to_num(rows[..., 2], nan=0.0).sum(0)
    best = []
    for i in range(shape[0]):
        cand = [(-float(rows[r, i, 3 + j]), int(rows[r, i, 3 + top + j])) for r in range(blocks.shape[0]) for j in range(top)
                if float(rows[r, i, 3 + j]) > -torch.inf]
        best.append([c[1] for c in sorted(cand)[:top]])
    return (xt - total.log()).tolist(), (total.log() - rows[..., 1].sum(0) / total).tolist(), best


def _w_logprobs(rank, world, v):
    import torch.distributed as dist

    from minitp_b200.distributed.context import ParallelContext
    from minitp_b200.parallel import embedding

    embedding.ops.logprobs_block, embedding.ops.logprobs_join = _cpu_block, _cpu_join
    head = embedding.VocabParallelLMHead(8, v, ParallelContext(rank, rank, world, rank, world, torch.device("cpu"), dist.group.WORLD))
    x, t = _logprob_case(v)
    return head.token_logprobs(x[:, head.vocab_start:head.vocab_end], t, 4)


def _logprob_case(v):
    r = torch.Generator().manual_seed(v)
    return torch.randn(5, v, generator=r), torch.randint(0, v, (5,), generator=r)


@pytest.mark.distributed
@pytest.mark.parametrize("world,v", [(2, 101), (3, 10), (3, 5)])
def test_logprobs_exchange_the_shards_of_all_ranks(world, v):
    """`VocabParallelLMHead.token_logprobs` over Gloo ranks (the kernels played by the stand-ins above): every rank
    gets the whole vocabulary's values, of uneven shards too."""
    from tests.tp_harness import run_tp

    x, t = _logprob_case(v)
    lp = torch.log_softmax(x.double(), -1)
    res = run_tp(world, _w_logprobs, v)
    for r in range(world):
        got, ent, best = res[r]
        assert got == pytest.approx(lp.gather(1, t[:, None])[:, 0].tolist(), abs=1e-9)
        assert ent == pytest.approx((-(lp.exp() * lp).sum(-1)).tolist(), abs=1e-9)
        assert best == lp.topk(min(4, v), dim=-1).indices.tolist()



def _w_score(rank, world, v):
    from types import SimpleNamespace

    import torch.distributed as dist

    from minitp_b200 import scoring
    from minitp_b200.distributed.context import ParallelContext
    from minitp_b200.parallel import embedding

    embedding.ops.logprobs_block = _cpu_block
    embedding.ops.logprobs_join = lambda *a: tuple(torch.tensor(x) for x in _cpu_join(*a)) + (None,)
    embedding.ops.linear = torch.nn.functional.linear
    scoring._LOGITS_BYTES = 1000  # 4 rows of the larger shard, 5 of the smaller one
    table, weight = _score_case(v)
    head = embedding.VocabParallelLMHead(8, v, ParallelContext(rank, rank, world, rank, world, torch.device("cpu"), dist.group.WORLD))
    head.weight.data = weight[head.vocab_start:head.vocab_end]
    model = SimpleNamespace(model=SimpleNamespace(embed_tokens=SimpleNamespace(weight=table)), lm_head=head,
                            cfg=SimpleNamespace(max_position_embeddings=64, vocab_size=v),
                            forward_packed=lambda ids, starts: table[ids])
    return [s.logprobs.tolist() for s in scoring.score_prompts(model, [[3, 1, 4, 1, 5, 9, 2], [6], [5, 3, 5, 8, 9]])]


def _score_case(v):
    r = torch.Generator().manual_seed(v)
    return torch.randn(v, 8, generator=r), torch.randn(v, 8, generator=r)


@pytest.mark.distributed
def test_ranks_with_uneven_shards_score_in_the_same_pieces(lib):
    """Every rank cuts the tokens into the same pieces, whatever its share of the vocabulary (the kernels played by
    stand-ins, the hidden states by a table)."""
    from tests.tp_harness import run_tp

    table, weight = _score_case(101)
    want = []
    for ids in ([3, 1, 4, 1, 5, 9, 2], [6], [5, 3, 5, 8, 9]):
        lp = torch.log_softmax((table[ids[:-1]] @ weight.T).double(), -1)
        want.append([float(lp[i, t]) for i, t in enumerate(ids[1:])])
    for got in run_tp(2, _w_score, 101).values():
        for g, w in zip(got, want):
            assert g == pytest.approx(w, abs=1e-4)  # (fp32 logits of magnitude 10 to 20, their log-sum in 64 bits)


def test_packed_forward_refusals(lib):
    ok = dict(model=P, ids=P, T=4, pos=P, starts=P, S=1, k=P, v=P, hidden=P, st=None)
    # (a model's own sizes are looked at only after these)
    for change, match in [(dict(model=None), "null"), (dict(ids=None), "null"), (dict(pos=None), "null"), (dict(starts=None), "null"),
                          (dict(hidden=None), "null"), (dict(k=None), "null"), (dict(T=0), "empty"), (dict(S=-1), "empty")]:
        _refused(lib, "mtpb_model_forward_packed", list((ok | change).values()), match)


def test_prompts_that_are_no_integers_are_refused():
    """Lists are held to what tensors are: nothing is cut to an integer on the way (before any use of the model)."""
    from types import SimpleNamespace

    import numpy as np

    from minitp_b200 import scoring

    model = SimpleNamespace(model=SimpleNamespace(embed_tokens=SimpleNamespace(weight=torch.zeros(1))),
                            cfg=SimpleNamespace(max_position_embeddings=64, vocab_size=10))
    for wrong in ([1.5, 2], [1.0, 2.0], np.array([1.0, 2.0]), "12", [[1, 2], [3, 4]], [1, None], [2 ** 70], torch.zeros(2)):
        with pytest.raises(ValueError, match="sequences"):
            scoring.score_prompts(model, [[1, 2], wrong])
    for fine in ([1, 2], (1, 2), np.array([1, 2]), np.array([1, 2], dtype=np.uint16), range(1, 3), [torch.tensor(1), np.int32(2)]):
        assert scoring._id_tensor(fine).tolist() == [1, 2]
    assert scoring._id_tensor([]).dtype == torch.int64
