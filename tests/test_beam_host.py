"""Refusals of the beam-search and shared-prefix calls (host checks; no GPU, no launch)."""

import ctypes

import pytest
import torch

from minitp_b200 import _lib, ops

P = 1 << 20  # a 16-byte aligned stand-in for a device address; every call below is refused before it is used


def _refused(lib, name, args, match):
    assert getattr(lib, name)(*args) == _lib.ERR_INVALID
    assert match in lib.mtpb_last_error().decode()


def test_select_refusals(lib):
    ok = dict(logits=P, ld=100, G=2, W=4, V=100, scores=P, finished=None, eos=-1, k=4, o=P, p=P, t=P, f=None, block=P,
              dtype=_lib.MTPB_F32, st=None)
    for change, match in [(dict(logits=None), "null"), (dict(scores=None), "null"), (dict(k=0), "k must"),
                          (dict(k=65), "k must"), (dict(W=65), "64 beams"), (dict(W=0), "64 beams"),
                          (dict(G=0), "64 beams"), (dict(V=0), "vocabulary"), (dict(ld=99), "ld"),
                          (dict(dtype=7), "dtype"), (dict(block=P + 8), "aligned"), (dict(finished=P), "end token"),
                          (dict(eos=2 ** 32), "end token"), (dict(o=None), "null"), (dict(G=40000), "65535")]:
        _refused(lib, "mtpb_beam_select", list((ok | change).values()), match)
    assert lib.mtpb_beam_block_bytes(8, 151936, 65) < 0
    assert lib.mtpb_beam_block_bytes(1, 2 ** 30 - 1, 4) > 0 > lib.mtpb_beam_block_bytes(1, 2 ** 30, 4)
    assert lib.mtpb_beam_block_bytes(0, 151936, 4) < 0
    assert lib.mtpb_beam_block_bytes(8, 151936, 4) > 0


def test_candidates_and_pick_refusals(lib):
    ok = dict(logits=P, ld=50, rows=8, v=50, vstart=0, plan=60, k=4, finished=None, block=P, dtype=_lib.MTPB_BF16, st=None)
    for change, match in [(dict(v=61), "V_plan"), (dict(v=-1), "V_plan"), (dict(vstart=-1), "range"),
                          (dict(vstart=2 ** 32), "range"), (dict(block=None), "null"), (dict(rows=0), "rows")]:
        _refused(lib, "mtpb_beam_candidates", list((ok | change).values()), match)
    ok = dict(blocks=P, parts=2, G=2, W=4, plan=60, kb=4, scores=P, finished=None, eos=-1, k=4, o=P, p=P, t=P, f=None,
              st=None)
    for change, match in [(dict(parts=0), "shards"), (dict(parts=65), "shards"), (dict(k=5), "blocks' k"),
                          (dict(blocks=None), "aligned"), (dict(scores=None), "null"), (dict(kb=0), "k must")]:
        _refused(lib, "mtpb_beam_pick", list((ok | change).values()), match)


def test_one_limit_of_rows(lib):
    """A block can be sized for just the rows that the selection and its halves take."""
    assert lib.mtpb_beam_block_bytes(65535, 1000, 4) > 0
    for rows in (65536, 1 << 20, (1 << 20) + 1):
        assert lib.mtpb_beam_block_bytes(rows, 1000, 4) == _lib.ERR_INVALID
        assert "65535" in lib.mtpb_last_error().decode()
    _refused(lib, "mtpb_beam_candidates", (P, 50, 65536, 50, 0, 60, 4, None, P, _lib.MTPB_BF16, None), "65535")
    _refused(lib, "mtpb_beam_pick", (P, 2, 1024, 64, 60, 4, P, None, -1, 4, P, P, P, None, None), "65535")
    _refused(lib, "mtpb_beam_select", (P, 100, 1024, 64, 100, P, None, -1, 4, P, P, P, None, P, _lib.MTPB_F32, None), "65535")


def test_reorder_refusals(lib):
    arr = (ctypes.c_void_p * 2)(P, P)
    odd = (ctypes.c_void_p * 2)(P, P + 8)
    none = (ctypes.c_void_p * 2)(P, None)
    ok = dict(k=arr, v=arr, n=2, parents=P, lens=None, len=5, G=1, W=4, hkv=2, cap=8, hd=64, dtype=_lib.MTPB_BF16, st=None)
    for change, match in [(dict(k=None), "null"), (dict(parents=None), "null"), (dict(n=0), "positive"),
                          (dict(W=65), "64 rows"), (dict(len=9), "outside"), (dict(len=-1), "outside"),
                          (dict(hd=4), "16 bytes"), (dict(k=odd), "aligned"), (dict(v=none), "aligned"),
                          (dict(G=70000), "65535"), (dict(dtype=3), "dtype")]:
        _refused(lib, "mtpb_kv_reorder", list((ok | change).values()), match)


def test_reorder_refuses_caches_that_overlap(lib):
    size = 4 * 2 * 8 * 64 * 2  # bytes of a cache
    for ks, vs in [((P, P + size), (P + 2 * size, P)), ((P, P + size - 16), (P + 4 * size, P + 8 * size)), ((P,), (P,))]:
        n = len(ks)
        arr = ctypes.c_void_p * n
        _refused(lib, "mtpb_kv_reorder", (arr(*ks), arr(*vs), n, P, None, 5, 1, 4, 2, 8, 64, _lib.MTPB_BF16, None), "overlap")


def test_attention_refusals(lib):
    ok = dict(q=P, kp=P, vp=P, pl=None, plen=1 << 20, kc=P, vc=P, cl=None, clen=5, out=P, G=2, W=4, T=1, hq=14, hkv=2, hd=64,
              cap_p=1 << 20, cap=8, dtype=_lib.MTPB_BF16, ws=P, n=1 << 30, st=None)
    for change, match in [(dict(q=None), "null"), (dict(ws=None), "null"), (dict(n=16), "workspace"),
                          (dict(hd=80), "head_dim"), (dict(hkv=4), "multiple"), (dict(T=0), "positive"),
                          (dict(cap=0), "positive"), (dict(plen=(1 << 20) + 1), "prefix length"), (dict(plen=-1), "prefix length"),
                          (dict(clen=9), "length outside"), (dict(kp=P + 2), "aligned"), (dict(dtype=9), "dtype"),
                          (dict(G=1 << 20, W=1 << 10), "rows")]:
        _refused(lib, "mtpb_shared_attention", list((ok | change).values()), match)
    assert lib.mtpb_shared_attention_workspace(2, 4, 1, 14, 3, 64, 8, 8, 1) < 0


def _cpu_candidates(local_logits, k, vstart, v_plan, finished=None):
    """A stand-in for a shard's block: its best values with their ids and its sum of exponentials, as bytes."""
    g, w, v = local_logits.shape
    assert v <= v_plan
    x = torch.full((g, w, v_plan), -torch.inf, dtype=torch.float64)
    x[:, :, :v] = local_logits.double()
    val, at = torch.cat([x, torch.full((g, w, k), -torch.inf, dtype=torch.float64)], -1).sort(dim=-1, descending=True, stable=True)
    lse = torch.logsumexp(x, -1, keepdim=True)
    return torch.cat([val[..., :k], (at[..., :k] + vstart).double(), lse], -1).reshape(-1).view(torch.uint8)


def _cpu_pick(blocks, scores, k, v_plan, finished=None, eos_token_id=None):
    g, w = scores.shape
    rows = blocks.contiguous().view(torch.float64).view(blocks.shape[0], g, w, 2 * k + 1)
    lse = torch.logsumexp(rows[..., -1], 0)
    total = rows[..., :k] - lse[..., None] + scores.double()[..., None]
    best = []
    for i in range(g):
        cand = [(-float(total[r, i, b, j]), b, int(rows[r, i, b, k + j])) for r in range(blocks.shape[0]) for b in range(w)
                for j in range(k) if float(total[r, i, b, j]) > -torch.inf]
        best.append(sorted(cand)[:k])
    return [[(round(-s, 9), b, t) for s, b, t in row] for row in best]


def _w_beam_select(rank, world, v):
    import torch.distributed as dist

    from minitp_b200.distributed.context import ParallelContext
    from minitp_b200.parallel import embedding

    embedding.ops.beam_candidates, embedding.ops.beam_pick = _cpu_candidates, _cpu_pick
    head = embedding.VocabParallelLMHead(8, v, ParallelContext(rank, rank, world, rank, world, torch.device("cpu"), dist.group.WORLD))
    x, s = _beam_case(v)
    return head.beam_select(x[:, :, head.vocab_start:head.vocab_end], s, 4)


def _beam_case(v):
    r = torch.Generator().manual_seed(v)
    return torch.randn(2, 3, v, generator=r), torch.randn(2, 3, generator=r)


@pytest.mark.distributed
@pytest.mark.parametrize("world,v", [(2, 101), (3, 10), (3, 2)])
def test_selection_exchanges_the_shards_of_all_ranks(world, v):
    """`VocabParallelLMHead.beam_select` over Gloo ranks (the kernels played by the stand-ins above): every rank gets
    the whole vocabulary's candidates, of uneven and empty shards too."""
    from tests.tp_harness import run_tp

    res = run_tp(world, _w_beam_select, v)
    x, s = _beam_case(v)
    total = (s.double()[..., None] + torch.log_softmax(x.double(), -1)).view(2, -1)
    val, at = total.sort(dim=-1, descending=True, stable=True)
    n = min(4, 3 * v)
    want = [[(round(float(a), 9), int(b) // v, int(b) % v) for a, b in zip(val[i, :n], at[i, :n])] for i in range(2)]
    for r in range(world):
        assert [[c[1:] for c in row] for row in res[r]] == [[c[1:] for c in row] for row in want]
        assert [c[0] for row in res[r] for c in row] == pytest.approx([c[0] for row in want for c in row], abs=1e-8)


def test_cpu_tensors_are_refused(lib):
    with pytest.raises(_lib.MinitpB200Error, match="CUDA"):
        ops.beam_select(torch.zeros(1, 2, 10), torch.zeros(1, 2), 2)
    with pytest.raises(_lib.MinitpB200Error, match="CUDA"):
        ops.reorder_cache_([torch.zeros(2, 1, 4, 16)], [torch.zeros(2, 1, 4, 16)], torch.zeros(1, 2, dtype=torch.long), 4)
    c = torch.zeros(2, 1, 4, 16)
    with pytest.raises(_lib.MinitpB200Error, match="CUDA"):
        ops.shared_prefix_attention(torch.zeros(2, 1, 32), c, c, 4, c, c, 4, 2, 1)


def test_shapes_and_types_are_refused(lib):
    x, s = torch.zeros(1, 2, 10), torch.zeros(1, 2)
    with pytest.raises(_lib.MinitpB200Error, match="need logits"):
        ops.beam_select(x[0], s, 2)
    with pytest.raises(_lib.MinitpB200Error, match="need logits"):
        ops.beam_select(x, s[:, :1], 2)
    with pytest.raises(_lib.MinitpB200Error, match="as many K as V"):
        ops.reorder_cache_([x], [], torch.zeros(1, 2, dtype=torch.long), 4)
    with pytest.raises(_lib.MinitpB200Error, match="int64"):
        ops.reorder_cache_([x], [x], torch.zeros(1, 2), 4)
