"""Beam selection, cache reordering and shared-prefix attention against plain 64-bit implementations."""

import math

import pytest
import torch

from tests import beam_ref

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------ selection
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("g,w,v,k", [(1, 1, 1, 1), (1, 4, 1000, 4), (2, 3, 7, 5), (3, 8, 5000, 8), (1, 4, 151936, 4),
                                     (2, 1, 151937, 64), (1, 64, 333, 64), (5, 5, 4097, 10), (1, 2, 8192, 33),
                                     (40, 2, 20001, 4), (2, 2, 31, 64)])
def test_select(lib, dtype, g, w, v, k):
    from minitp_b200 import ops

    r = _gen(g * 1000 + w * 100 + v + k)
    x = (torch.randn(g, w, v, generator=r) * 3).to(DT[dtype])
    s = torch.randn(g, w, generator=r) * 2 - 20
    got = ops.beam_select(x.cuda(), s.cuda(), k)
    beam_ref.check_select(got, x, s, k)
    fin = torch.rand(g, w, generator=r) < 0.4
    got = ops.beam_select(x.cuda(), s.cuda(), k, fin.cuda(), v // 2)
    beam_ref.check_select(got, x, s, k, fin, v // 2)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_select_ties_go_to_the_lowest_index(lib, dtype):
    from minitp_b200 import ops

    for v, k in [(20, 6), (9000, 16), (30000, 64)]:
        x = torch.zeros(1, 3, v, dtype=DT[dtype])
        x[0, 2, 5] = -0.0  # the same value as +0.0
        s = torch.zeros(1, 3)
        out, par, tok, _ = ops.beam_select(x.cuda(), s.cuda(), k)
        flat = (par * v + tok).cpu()[0].tolist()
        assert flat == list(range(k))
        assert float((out.cpu().double() + math.log(v)).abs().max()) <= beam_ref.select_tolerance(v, out.cpu().double())
        # few distinct values: long runs of equal logits across chunk borders
        y = torch.randint(0, 3, (1, 3, v), generator=_gen(v)).to(DT[dtype])
        s = torch.tensor([[-1.0, -1.5, -9.0]])
        beam_ref.check_select(ops.beam_select(y.cuda(), s.cuda(), k), y, s, k)


def test_select_masks_infinities_and_nan(lib):
    from minitp_b200 import ops

    inf, nan = math.inf, math.nan
    lowest = torch.finfo(torch.float32).min
    x = torch.full((4, 3, 40), -inf)
    x[0, 0, :3] = torch.tensor([1.0, nan, 2.0])  # a banned token by NaN
    x[0, 1, 7] = 0.5  # one token left; beam 2 has none
    x[1, 0, 4:6] = inf  # two +inf tokens share the probability
    x[1, 0, 8] = 3.0
    x[1, 1] = lowest  # masked by the type's lowest value: a uniform row
    x[1, 2] = nan
    x[2] = torch.randn(3, 40, generator=_gen(1))
    s = torch.tensor([[-1.0, -2.0, 0.0], [-1.0, -2.0, -3.0], [-inf, nan, -4.0], [0.0, 0.0, 0.0]])
    for k in (1, 3, 8, 50):
        beam_ref.check_select(ops.beam_select(x.cuda(), s.cuda(), k), x, s, k)
    out, par, tok, _ = ops.beam_select(x.cuda(), s.cuda(), 4)
    assert out[3].tolist() == [-inf] * 4 and par[3].tolist() == [0] * 4 and tok[3].tolist() == [0] * 4
    assert out[1, 0].item() == pytest.approx(-1 - math.log(2), abs=1e-6) and tok[1, :2].tolist() == [4, 5]
    fin = torch.tensor([[False, True, True]] * 4)
    for k in (1, 3, 8):
        beam_ref.check_select(ops.beam_select(x.cuda(), s.cuda(), k, fin.cuda(), 39), x, s, k, fin, 39)
    y = x.to(torch.bfloat16)  # the lowest fp32 value becomes -inf there
    beam_ref.check_select(ops.beam_select(y.cuda(), s.cuda(), 8), y, s, 8)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("mask", [-1e4, -1e9, -1e10, -3e10, -1e11, -1e12, -1e20, 1e4, 1e6, 1e9, 1e10, 1e12, 1e20])
@pytest.mark.parametrize("v", [40, 30000])
def test_select_logits_far_from_zero(lib, dtype, mask, v):
    """Banned tokens of any large value beside a few live ones, and rows that hold nothing else."""
    from minitp_b200 import ops

    r = _gen(v + int(abs(mask)) % 1000)
    x = torch.full((3, 3, v), mask)
    live = torch.randint(0, v, (3, 3, 5), generator=r)
    x.scatter_(2, live, torch.randn(3, 3, 5, generator=r) * 3)
    x[1, 0] = mask  # one such row beside others
    x[2, 1:] = mask
    x[2, 0] = torch.randn(v, generator=r) * 3  # .. and beside a plain one
    x = x.to(DT[dtype])
    s = torch.randn(3, 3, generator=r) * 2 - 20
    for k in (1, 3, 8, 24):
        beam_ref.check_totals(ops.beam_select(x.cuda(), s.cuda(), k), x, s, k)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("v", [333, 20001])
def test_select_logits_of_every_size(lib, dtype, v):
    """Rows moved away from zero, rows of every spread, and logits around the border from which on equal
    values are counted (2^30), where neighbours are 64 and 128 apart."""
    from minitp_b200 import ops

    r = _gen(v)
    rows = [torch.randn(v, generator=r) * 3 + d for d in (-1e4, 1e4, -1e6, 1e6, 3e7, -3e8)]
    rows += [torch.randn(v, generator=r) * 10.0 ** e for e in range(1, 16)]
    border = 2.0 ** 30
    steps = torch.tensor([-192.0, -128.0, -64.0, 0.0, 128.0, 256.0])
    rows += [sign * (border + steps[torch.randint(0, n, (v,), generator=r)]) for n in (3, 4, 6) for sign in (1, -1)]
    rows += [(border / 2 + steps[torch.randint(0, 6, (v,), generator=r)] / 2) * sign for sign in (1, -1)]
    rows += [-(border + 64.0 * torch.randint(-8, 9, (v,), generator=r)), torch.full((v,), -border), torch.full((v,), border - 64)]
    x = torch.stack(rows)[:, None].to(DT[dtype])
    s = torch.randn(len(rows), 1, generator=r)
    for k in (1, 9):
        beam_ref.check_totals(ops.beam_select(x.cuda(), s.cuda(), k), x, s, k)
    # pairs of such rows as the beams of one prompt
    n = len(rows) // 2 * 2
    x, s = x[:n].reshape(n // 2, 2, v), s[:n].reshape(n // 2, 2)
    beam_ref.check_totals(ops.beam_select(x.cuda(), s.cuda(), 9), x, s, 9)


def test_select_first_step_from_one_beam(lib):
    """The first step: one live beam per prompt gives k different tokens."""
    from minitp_b200 import ops

    x = torch.randn(2, 1, 999, generator=_gen(3))
    s = torch.zeros(2, 1)
    out, par, tok, _ = ops.beam_select(x.cuda(), s.cuda(), 8)
    want = torch.log_softmax(x.double(), -1)[:, 0].topk(8)
    assert torch.equal(tok.cpu(), want.indices) and int(par.sum()) == 0
    # the same from 8 beams of which one is in use
    x8 = x.expand(2, 8, 999).contiguous()
    s8 = torch.full((2, 8), -math.inf)
    s8[:, 0] = 0
    again = ops.beam_select(x8.cuda(), s8.cuda(), 8)
    assert torch.equal(again[2], tok) and torch.equal(again[0], out)


def test_select_strides(lib):
    from minitp_b200 import ops

    r = _gen(5)
    big = torch.randn(6, 4, 1013, generator=r).cuda()
    s = torch.randn(6, 4, generator=r).cuda()
    views = [big[:, :, 3:1000], big[:, :, 1:2], big[:, ::2, :800], big[::2], big.transpose(0, 1)[:, :4],
             big[:1, :1].expand(6, 4, 1013), big[:, 1:2], big[2:3, :, 5:]]
    for x in views:
        sc = s[: x.shape[0], : x.shape[1]].contiguous()
        beam_ref.check_select(ops.beam_select(x, sc, 4), x, sc, 4)
    xb = torch.randn(3, 2, 2051, generator=r).to(torch.bfloat16).cuda()[:, :, 1:]  # rows off every vector border
    beam_ref.check_select(ops.beam_select(xb, s[:3, :2].contiguous(), 7), xb, s[:3, :2], 7)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("parts,v", [(2, 151937), (3, 10), (8, 4099), (4, 3)])
def test_select_from_vocabulary_shards(lib, dtype, parts, v):
    """Candidates of uneven shards, picked together, are the selection over the whole vocabulary."""
    from minitp_b200 import ops
    from minitp_b200.parallel.linear import shard_range

    r = _gen(v)
    g, w, k, eos = 2, 4, 8, 1
    x = (torch.randn(g, w, v, generator=r) * 2).to(DT[dtype]).cuda()
    s = torch.randn(g, w, generator=r).cuda()
    fin = (torch.rand(g, w, generator=r) < 0.3).cuda()
    plan = -(-v // parts)
    blocks = []
    for p in range(parts):
        a, b = shard_range(v, p, parts)
        blocks.append(ops.beam_candidates(x[:, :, a:b], k, a, plan, fin))
    got = ops.beam_pick(torch.stack(blocks), s, k, plan, fin, eos)
    beam_ref.check_select(got, x, s, k, fin, eos)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("tp,v", [(2, 1001), (3, 4099), (8, 11)])
def test_select_by_the_ranks_of_a_vocabulary(lib, monkeypatch, dtype, tp, v):
    """`VocabParallelLMHead.beam_select` of every rank, one after the other with the exchange played by the test: the
    same places on all of them, those of the whole vocabulary."""
    from minitp_b200 import ops
    from minitp_b200.distributed.context import ParallelContext
    from minitp_b200.parallel import embedding

    r = _gen(v + tp)
    g, w, k, eos = 3, 4, 4, v - 1
    x = (torch.randn(g, w, v, generator=r) * 2).to(DT[dtype]).cuda()
    s = torch.randn(g, w, generator=r).cuda()
    fin = (torch.rand(g, w, generator=r) < 0.3).cuda()
    heads = [embedding.VocabParallelLMHead(8, v, ParallelContext(i, i, tp, i, tp, torch.device("cuda"), None)) for i in range(tp)]
    shards = [x[:, :, h.vocab_start:h.vocab_end].contiguous() for h in heads]
    sent: dict = {}

    class Sent(Exception):
        pass

    def send(out, mine, group):
        assert out.shape == (tp, mine.numel()) and out.dtype == mine.dtype
        sent[len(sent)] = mine
        raise Sent

    monkeypatch.setattr(embedding, "all_gather_dim0", send)
    for h, part in zip(heads, shards):
        with pytest.raises(Sent):
            h.beam_select(part, s, k, fin, eos)
    assert len({b.numel() for b in sent.values()}) == 1
    monkeypatch.setattr(embedding, "all_gather_dim0", lambda out, mine, group: out.copy_(torch.stack(list(sent.values()))))
    got = [h.beam_select(part, s, k, fin, eos) for h, part in zip(heads, shards)]
    whole = ops.beam_select(x, s, k, fin, eos)
    for o in got:
        assert all(torch.equal(a, b) for a, b in zip(o, got[0]))
        assert all(torch.equal(a, b) for a, b in zip(o[1:], whole[1:]))  # (scores: chunks are cut elsewhere)
    beam_ref.check_select(got[0], x, s, k, fin, eos)


def test_select_streams_and_graph(lib):
    """Two calls at once on two streams, and a captured call replayed on new inputs."""
    from minitp_b200 import ops

    r = _gen(9)
    xs = [torch.randn(4, 4, 30000, generator=r).cuda() for _ in range(2)]
    s = torch.randn(4, 4, generator=r).cuda()
    want = [ops.beam_select(x, s, 4) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for st, x in zip(streams, xs):
            with torch.cuda.stream(st):
                got.append(ops.beam_select(x, s, 4))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(o[:3], want[i % 2][:3]))
    x = xs[0].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = ops.beam_select(x, s, 4)
    for i in (1, 0, 1):
        x.copy_(xs[i])
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(o[:3], want[i][:3]))


# ------------------------------------------------------------------ reordering
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("layers,g,w,hkv,hd,cap", [(1, 1, 1, 1, 16, 4), (2, 1, 4, 2, 16, 9), (3, 2, 8, 1, 64, 33),
                                                   (2, 3, 5, 4, 128, 17), (1, 1, 16, 2, 64, 40), (70, 1, 3, 1, 16, 5),
                                                   (2, 1, 27, 2, 32, 12), (1, 2, 64, 1, 128, 7)])
def test_reorder(lib, dtype, layers, g, w, hkv, hd, cap):
    from minitp_b200 import ops

    r = _gen(layers * 100 + w)
    mk = lambda: [torch.randn(g * w, hkv, cap, hd, generator=r).to(DT[dtype]) for _ in range(layers)]  # noqa: E731
    for parents in (torch.randint(0, w, (g, w), generator=r), torch.arange(w).flip(0).repeat(g, 1),
                    torch.arange(w).roll(1).repeat(g, 1), torch.zeros(g, w, dtype=torch.int64),
                    torch.arange(w).repeat(g, 1)):
        for lengths in (torch.randint(0, cap + 1, (g * w,), generator=r, dtype=torch.int32), cap, 0, 1):
            k, v = mk(), mk()
            kg, vg = [t.cuda() for t in k], [t.cuda() for t in v]
            ops.reorder_cache_(kg, vg, parents.cuda(), lengths if isinstance(lengths, int) else lengths.cuda())
            ln = [lengths] * (g * w) if isinstance(lengths, int) else lengths
            for a, b in zip(kg + vg, k + v):
                assert torch.equal(a.cpu(), beam_ref.reorder(b, parents, ln))


def test_reorder_leaves_rows_of_parents_out_of_range(lib):
    from minitp_b200 import ops

    k, v = (torch.randn(4, 1, 6, 16).cuda() for _ in range(2))
    k0, v0 = k.clone(), v.clone()
    parents = torch.tensor([[1, -1, 4, 2 ** 40]]).cuda()
    lens = torch.tensor([3, 100, -5, 6], dtype=torch.int32).cuda()  # clamped to the cache
    ops.reorder_cache_([k], [v], parents, lens)
    k0[0], v0[0] = k0[1], v0[1]
    assert torch.equal(k, k0) and torch.equal(v, v0)


def test_reorder_in_a_graph(lib):
    from minitp_b200 import ops

    r = _gen(2)
    src = [torch.randn(8, 2, 20, 64, generator=r).cuda() for _ in range(4)]
    k, v = [t.clone() for t in src[:2]], [t.clone() for t in src[2:]]
    parents = torch.arange(4).repeat(2, 1).cuda()
    lens = torch.full((8,), 20, dtype=torch.int32).cuda()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.reorder_cache_(k, v, parents, lens)
    for seed in (3, 4):
        parents.copy_(torch.randint(0, 4, (2, 4), generator=_gen(seed)))
        lens.fill_(seed * 4)
        for a, b in zip(k + v, src):
            a.copy_(b)
        g.replay()
        for a, b in zip(k + v, src):
            assert torch.equal(a.cpu(), beam_ref.reorder(b.cpu(), parents.cpu(), lens.cpu()))


# ------------------------------------------------------------------ attention
def _attention_case(seed, dtype, g, w, t, hq, hkv, hd, cap_p, plens, cap, clens, poison=math.nan):
    r = _gen(seed)
    dt = DT[dtype]
    q = (torch.randn(g * w, t, hq * hd, generator=r) * 1.5).to(dt)
    kp, vp = (torch.randn(g, hkv, cap_p, hd, generator=r).to(dt) for _ in range(2))
    kc, vc = (torch.randn(g * w, hkv, cap, hd, generator=r).to(dt) for _ in range(2))
    for i, n in enumerate(plens):  # what lies behind the last position is never used
        kp[i, :, max(0, n):] = poison
        vp[i, :, max(0, n):] = poison
    for i, n in enumerate(clens):
        kc[i, :, max(0, n):] = poison
        vc[i, :, max(0, n):] = poison
    return q, kp, vp, torch.tensor(plens, dtype=torch.int32), kc, vc, torch.tensor(clens, dtype=torch.int32)


def _check_attention(case, hq, hkv):
    from minitp_b200 import ops

    got = ops.shared_prefix_attention(*(x.cuda() for x in case), hq, hkv).cpu()
    want, tol = beam_ref.attend(*case, hq, hkv)
    assert got.dtype == case[0].dtype
    off = (got.double() - want).abs()
    assert torch.isfinite(got.float()).all()
    assert bool((off <= tol).all()), float((off - tol).max())
    return got


HEADS = [(4, 2, 16), (8, 4, 32), (14, 2, 64), (7, 1, 128), (28, 4, 128), (4, 1, 128), (3, 3, 64), (20, 1, 64)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("hq,hkv,hd", HEADS)
@pytest.mark.parametrize("g,w,plens,clens", [
    (1, 1, [1], [1]),
    (1, 4, [128], [16] * 4),
    (2, 3, [65, 200], [0, 1, 2, 63, 64, 65]),
    (3, 2, [0, 1, 513], [0, 5, 0, 130, 129, 0]),
])
def test_attention_single_tokens(lib, dtype, hq, hkv, hd, g, w, plens, clens):
    case = _attention_case(hq * hd + g + w, dtype, g, w, 1, hq, hkv, hd, max(plens) + 3, plens, max(clens) + 2, clens)
    got = _check_attention(case, hq, hkv)
    for r in range(g * w):
        if plens[r // w] == 0 and clens[r] == 0:
            assert int((got[r] != 0).sum()) == 0  # nothing seen: zeros


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("hq,hkv,hd", [(4, 2, 16), (14, 2, 64), (7, 1, 128)])
@pytest.mark.parametrize("g,w,t,plens,clens", [
    (1, 2, 5, [70], [5, 9]),
    (2, 2, 19, [0, 33], [19, 25, 40, 3]),  # fewer own positions than tokens: the first tokens see only the prefix
    (1, 1, 140, [129], [140]),
    (2, 1, 33, [300, 0], [0, 60]),
])
def test_attention_many_tokens(lib, dtype, hq, hkv, hd, g, w, t, plens, clens):
    case = _attention_case(hq + hd + t, dtype, g, w, t, hq, hkv, hd, max(plens) + 1, plens, max(clens) + 5, clens)
    _check_attention(case, hq, hkv)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_attention_wide_groups_and_long_prefixes(lib, dtype):
    # 40 rows x 7 heads fill more than two row tiles; the prefix ends inside a key tile
    case = _attention_case(1, dtype, 1, 40, 1, 7, 1, 128, 1500, [1333], 40, [i for i in range(40)])
    _check_attention(case, 7, 1)
    case = _attention_case(2, dtype, 2, 3, 1, 14, 2, 64, 5000, [4999, 2500], 700, [700, 1, 0, 333, 512, 640])
    _check_attention(case, 14, 2)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("hq,hkv,hd", [(14, 2, 64), (4, 1, 128), (40, 2, 128)])
def test_attention_long_own_caches_of_few_rows(lib, dtype, hq, hkv, hd):
    """Own caches cut into key ranges, behind no prefix, a short one and one of many ranges."""
    case = _attention_case(hq, dtype, 3, 1, 1, hq, hkv, hd, 3000, [0, 64, 2999], 2200, [2200, 700, 0])
    _check_attention(case, hq, hkv)
    case = _attention_case(hq + 1, dtype, 1, 2, 1, hq, hkv, hd, 1, [1], 4100, [4099, 1])
    _check_attention(case, hq, hkv)


def test_attention_large_scores_and_masked_infinities(lib):
    """Scores of hundreds (one key takes all), and infinities behind the last position."""
    for dtype in ("fp32", "bf16"):
        case = _attention_case(3, dtype, 1, 3, 1, 4, 2, 64, 200, [190], 30, [10, 0, 30], poison=math.inf)
        q = (case[0].float() * 40).to(DT[dtype])
        _check_attention((q, *case[1:]), 4, 2)


ODD_SIZES = [  # dtype, hq, hkv, hd, g, w, t: each kernel and tile
    ("fp32", 4, 2, 16, 1, 3, 1), ("fp32", 4, 1, 64, 1, 2, 5), ("fp32", 4, 1, 128, 1, 2, 70), ("bf16", 4, 2, 32, 1, 2, 20),
    ("bf16", 14, 2, 64, 1, 3, 1), ("bf16", 20, 1, 128, 1, 3, 1), ("bf16", 4, 2, 64, 1, 40, 1), ("bf16", 4, 2, 64, 1, 3, 5),
    ("bf16", 2, 1, 128, 1, 2, 60), ("bf16", 8, 1, 64, 1, 2, 40), ("bf16", 8, 1, 128, 1, 2, 150)]


@pytest.mark.parametrize("dtype,hq,hkv,hd,g,w,t", ODD_SIZES)
@pytest.mark.parametrize("odd", [math.nan, math.inf])
def test_attention_odd_values_stay_where_they_are_seen(lib, dtype, hq, hkv, hd, g, w, t, odd):
    """A value of an own V that is not finite reaches its dim of the tokens that see it, and nothing else."""
    from minitp_b200 import ops

    q, kp, vp, pl, kc, vc, cl = _attention_case(11, dtype, g, w, t, hq, hkv, hd, 300, [260] * g, t + 9, [t + 7] * (g * w))
    places = sorted({3, 7, 7 + t // 3, 6 + t})
    for n, j in enumerate(places):
        vc[1, hkv - 1, j, (5 + 9 * n) % hd] = odd
    got = ops.shared_prefix_attention(*(x.cuda() for x in (q, kp, vp, pl, kc, vc, cl)), hq, hkv).cpu()
    got = got.view(g * w, t, hq, hd).double()
    clean = vc.clone()
    clean[:, :, :t + 7][~torch.isfinite(vc[:, :, :t + 7])] = 0
    want, tol = (x.view(g * w, t, hq, hd) for x in beam_ref.attend(q, kp, vp, pl, kc, clean, cl, hq, hkv))
    reached = torch.zeros(got.shape, dtype=torch.bool)
    per = hq // hkv
    for n, j in enumerate(places):  # token i sees own positions [0, 8 + i)
        reached[1, max(0, j - 7):, (hkv - 1) * per:, (5 + 9 * n) % hd] = True
    assert torch.equal(~torch.isfinite(got), reached)
    assert bool(((got - want).abs() <= tol)[~reached].all())
    if odd == math.inf:
        assert bool((got[reached] == odd).all())


@pytest.mark.parametrize("dtype,hq,hkv,hd,g,w,t", ODD_SIZES)
def test_attention_nan_scores(lib, dtype, hq, hkv, hd, g, w, t):
    """A NaN in a query, or in a key that is seen, makes the rows NaN that score with it, and no other."""
    from minitp_b200 import ops

    q, kp, vp, pl, kc, vc, cl = _attention_case(12, dtype, g, w, t, hq, hkv, hd, 300, [260] * g, t + 9, [t + 7] * (g * w))
    per = hq // hkv
    clean = [x.clone() for x in (q, kp, vp, pl, kc, vc, cl)]
    want, tol = (x.view(g * w, t, hq, hd) for x in beam_ref.attend(*clean, hq, hkv))

    def check(case, reached):
        got = ops.shared_prefix_attention(*(x.cuda() for x in case), hq, hkv).cpu().view(g * w, t, hq, hd).double()
        assert torch.equal(got.isnan(), reached)
        assert bool(((got - want).abs() <= tol)[~reached].all())

    one = q.clone()
    one.view(g * w, t, hq, hd)[1, t // 2, 1, 3] = math.nan
    reached = torch.zeros(g * w, t, hq, hd, dtype=torch.bool)
    reached[1, t // 2, 1] = True
    check((one, kp, vp, pl, kc, vc, cl), reached)
    for j in (0, 2, 8, 5 + t):  # of the own cache of row 0
        one = kc.clone()
        one[0, 0, j, 1] = math.nan
        reached = torch.zeros(g * w, t, hq, hd, dtype=torch.bool)
        reached[0, max(0, j - 7):, :per] = True
        check((q, kp, vp, pl, one, vc, cl), reached)
    for j in (0, 128, 133, 259):  # of the prefix, which every row of the group sees
        one = kp.clone()
        one[0, 0, j, 1] = math.nan
        reached = torch.zeros(g * w, t, hq, hd, dtype=torch.bool)
        reached[:, :, :per] = True
        check((q, one, vp, pl, kc, vc, cl), reached)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("own", [False, True])
def test_attention_nan_beside_a_range_of_far_higher_scores(lib, hd, own):
    """A key range with a NaN score makes its rows NaN, however small its weight is in the join."""
    from minitp_b200 import ops

    n, t = (1, 40) if own else (40, 1)  # 160 rows of one KV head
    hq, hkv, long = 4, 1, 26000
    r = _gen(hd + own)
    u = torch.randn(hd, generator=r)
    u /= u.norm()
    q = (u * 20 + 0.1 * torch.randn(n, t, hq, hd, generator=r)).view(n, t, hq * hd)
    k, v = torch.randn(1, 1, long, hd, generator=r), torch.randn(1, 1, long, hd, generator=r)
    k[0, 0, 20000:20010] += u * 15 * math.sqrt(hd)  # scores of about 300; the others' are below 100
    small = torch.randn(1 if own else n, 1, t + 3, hd, generator=r)
    q, k, v, small = (x.to(torch.bfloat16).cuda() for x in (q, k, v, small))
    for j in (0, 1, 131, 4000, 19000):
        bad = k.clone()
        bad[0, 0, j, 3] = math.nan
        caches = (small, small, 0, bad, v, long) if own else (bad, v, long, small, small, t + 3)
        assert bool(ops.shared_prefix_attention(q, *caches, hq, hkv).isnan().all()), j


@pytest.mark.parametrize("odd", [math.nan, math.inf])
@pytest.mark.parametrize("dtype,hq,hkv,hd,g,w,t", ODD_SIZES)
def test_attention_odd_values_of_keys_that_weigh_nothing(lib, dtype, hq, hkv, hd, g, w, t, odd):
    """A NaN or an infinity among the V that a row sees reaches it from keys whose weight is below fp32's range too."""
    from minitp_b200 import ops

    r = _gen(hd + t)
    n, long = g * w, 26000 if t > 1 else 3000
    u = torch.randn(hd, generator=r)
    u /= u.norm()
    q = (u * 20 + 0.1 * torch.randn(n, t, hq, hd, generator=r)).view(n, t, hq * hd)
    kp, vp = (torch.randn(g, hkv, long, hd, generator=r) for _ in range(2))
    kc, vc = (torch.randn(n, hkv, 900 + t, hd, generator=r) for _ in range(2))
    high = u * 30 * math.sqrt(hd)  # scores of about 600; the others' are below 200
    kp[:, :, long - 9] += high
    kc[:, :, 899] += high  # (every token sees it)
    dev = [x.to(DT[dtype]).cuda() for x in (q, kp, vp, kc, vc)]
    for own, j in ((False, 2), (False, 133), (False, long // 2), (True, 1), (True, 17), (True, 40), (True, 700)):
        q_, kp_, vp_, kc_, vc_ = dev
        bad = (vc_ if own else vp_).clone()
        bad[0, hkv - 1, j, 5] = odd
        args = (q_, kp_, vp_, long, kc_, bad, 900 + t - 1) if own else (q_, kp_, bad, long, kc_, vc_, 900 + t - 1)
        got = ops.shared_prefix_attention(*args, hq, hkv).view(n, t, hq, hd)
        reached = torch.zeros(n, t, hq, hd, dtype=torch.bool)
        reached[: 1 if own else w, :, (hkv - 1) * (hq // hkv):, 5] = True
        assert torch.equal(~torch.isfinite(got.float().cpu()), reached), (own, j)
        if odd != odd:
            assert bool(got.cpu()[reached].isnan().all())


def test_attention_lengths_are_clamped_and_may_be_ints(lib):
    from minitp_b200 import ops

    q, kp, vp, pl, kc, vc, cl = (x.cuda() for x in _attention_case(4, "bf16", 2, 2, 1, 14, 2, 64, 50, [50, 50], 20,
                                                                   [20] * 4))
    want = ops.shared_prefix_attention(q, kp, vp, pl, kc, vc, cl, 14, 2)
    big = torch.tensor([51, 2 ** 30], dtype=torch.int32).cuda()
    assert torch.equal(ops.shared_prefix_attention(q, kp, vp, big, kc, vc, cl + 7, 14, 2), want)
    assert torch.equal(ops.shared_prefix_attention(q, kp, vp, 50, kc, vc, 20, 14, 2), want)
    none = ops.shared_prefix_attention(q, kp, vp, pl * 0 - 3, kc, vc, 0, 14, 2)
    assert int((none != 0).sum()) == 0


@pytest.mark.parametrize("t,hkv,hd,cap_p,plen,cap,clen", [
    (1, 2, 128, 9000, 7937, 1000, 151), (1, 1, 64, 9000, 5489, 1000, 271), (2, 2, 128, 9000, 6473, 300, 72)])
def test_attention_shorter_than_the_capacity(lib, t, hkv, hd, cap_p, plen, cap, clen):
    """Host lengths whose own plan would take more key ranges than the capacities' plan."""
    from minitp_b200 import ops

    q, kp, vp, pl, kc, vc, cl = _attention_case(9, "bf16", 1, 1, t, hkv, hkv, hd, cap_p, [plen], cap, [clen])
    want, tol = beam_ref.attend(q, kp, vp, pl, kc, vc, cl, hkv, hkv)
    got = ops.shared_prefix_attention(q.cuda(), kp.cuda(), vp.cuda(), plen, kc.cuda(), vc.cuda(), clen, hkv, hkv).cpu()
    assert bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_attention_of_more_rows_than_a_grid_axis(lib, dtype):
    from minitp_b200 import ops

    n, hd = 65539, 64
    r = _gen(13)
    q, kp, vp = (torch.randn(*s, generator=r).to(DT[dtype]) for s in ((n, 1, 2 * hd), (1, 1, 70, hd), (1, 1, 70, hd)))
    kc, vc = (torch.randn(n, 1, 6, hd, generator=r).to(DT[dtype]) for _ in range(2))
    cl = torch.randint(0, 7, (n,), generator=r, dtype=torch.int32)
    got = ops.shared_prefix_attention(*(x.cuda() for x in (q, kp, vp)), 65, kc.cuda(), vc.cuda(), cl.cuda(), 2, 1).cpu()
    some = torch.tensor([0, 1, 127, 128, 32768, 65534, 65535, 65536, n - 1])
    want, tol = beam_ref.attend(q[some], kp, vp, torch.tensor([65]), kc[some], vc[some], cl[some], 2, 1)
    assert bool(((got[some].double() - want).abs() <= tol).all())
    assert bool(torch.isfinite(got.float()).all())


def test_attention_equals_attention_over_one_cache(lib):
    """Prefix and own cache laid end to end give the framework's plain attention."""
    from minitp_b200 import ops

    for dtype in ("fp32", "bf16"):
        p, c = 300, 40
        case = _attention_case(6, dtype, 1, 4, 1, 14, 2, 64, p, [p], c, [c] * 4)
        q, kp, vp, pl, kc, vc, cl = (x.cuda() for x in case)
        got = ops.shared_prefix_attention(q, kp, vp, pl, kc, vc, cl, 14, 2)
        k = torch.cat([kp.expand(4, -1, -1, -1), kc], 2).contiguous()
        v = torch.cat([vp.expand(4, -1, -1, -1), vc], 2).contiguous()
        one = ops.attention(q, k, v, 14, 2, p + c - 1)
        want, tol = beam_ref.attend(*case, 14, 2)
        assert bool(((got.cpu().double() - want).abs() <= tol).all())
        assert bool(((one.cpu().double() - want).abs() <= tol).all())


def test_attention_streams_and_graph(lib):
    from minitp_b200 import ops

    cases = [[x.cuda() for x in _attention_case(s, "bf16", 1, 8, 1, 28, 4, 128, 700, [600], 64, [40] * 8)]
             for s in (1, 2)]
    want = [ops.shared_prefix_attention(*c, 28, 4) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for st, c in zip(streams, cases):
            with torch.cuda.stream(st):
                got.append(ops.shared_prefix_attention(*c, 28, 4))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 2])
    own = [x.clone() for x in cases[0]]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = ops.shared_prefix_attention(*own, 28, 4)
    for i in (1, 0, 1):
        for a, b in zip(own, cases[i]):
            a.copy_(b)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want[i])


def test_status_is_clean(lib):
    """No bounded wait of the calls above ran out."""
    import ctypes

    from minitp_b200 import _lib

    st = ctypes.c_uint32(7)
    _lib.call("mtpb_beam_status", ctypes.byref(st))
    assert st.value == 0


def test_refusals_before_a_launch(lib):
    """Arguments that the Python calls refuse for tensors on the device."""
    from minitp_b200 import _lib, ops

    def refused(match, call, *args):
        with pytest.raises(_lib.MinitpB200Error, match=match):
            call(*args)

    a, b = (torch.zeros(2, 1, 4, 16, device="cuda") for _ in range(2))
    parents = torch.zeros(1, 2, dtype=torch.long, device="cuda")
    refused("overlap", ops.reorder_cache_, [a, a], [b, b], parents, 4)
    refused("overlap", ops.reorder_cache_, [a], [a], parents, 4)
    for n in (5, -1, 2 ** 32 + 4):
        refused("outside", ops.reorder_cache_, [a], [b], parents, n)
    refused("lengths must", ops.reorder_cache_, [a], [b], parents, 4.0)
    refused("lengths must", ops.reorder_cache_, [a], [b], parents, torch.zeros(2, dtype=torch.long, device="cuda"))
    q = torch.zeros(2, 1, 32, device="cuda")
    c = torch.zeros(1, 1, 4, 16, device="cuda")
    refused("outside", ops.shared_prefix_attention, q, c, c, 2 ** 32, a, b, 4, 2, 1)
    refused("outside", ops.shared_prefix_attention, q, c, c, 4, a, b, 5, 2, 1)
    refused("do not fit", ops.shared_prefix_attention, q, c, c, 4, a, b, 4, 1, 1)
    refused("16-byte", ops.shared_prefix_attention, torch.zeros(65, device="cuda")[1:].view(2, 1, 32), c, c, 4, a, b, 4, 2, 1)
    x, s = torch.zeros(1, 2, 10, device="cuda"), torch.zeros(1, 2, device="cuda")
    refused("out of range", ops.beam_select, x, s, 2, None, 2 ** 32 - 1)
    refused("eos_token_id", ops.beam_select, x, s, 2, torch.zeros(1, 2, dtype=torch.bool, device="cuda"))
    refused("k in", ops.beam_select, x, s, 2 ** 32 + 2)
    refused("beam_candidates", ops.beam_candidates, x, 2, 2 ** 32, 10)
    refused("beam_candidates", ops.beam_candidates, x, 2, 0, 2 ** 32 + 10)
    refused("beam_candidates", ops.beam_candidates, x[0], 2, 0, 10)
    block = ops.beam_candidates(x, 2, 0, 10)
    refused("beam_pick", ops.beam_pick, block[None], s[0], 2, 10)
    refused("beam_pick", ops.beam_pick, block[None], s, 65, 10)
    refused("blocks must", ops.beam_pick, block[None], s, 3, 10)
