"""Beam search and decoding behind a shared prefix through the model, against plain CPU runs of the oracle model."""

import math

import pytest
import torch

from minitp_b200 import config as mcfg
from oracle.model import OracleConfig, OracleModel, checkpoint_tensors

pytestmark = pytest.mark.gpu

_CACHE: dict = {}


def _models(dtype=torch.float32):
    if dtype not in _CACHE:
        from minitp_b200.distributed.context import context_for
        from minitp_b200.weight_loader import load_synthetic_tp

        cfg = mcfg.baseline_tiny()
        gpu = load_synthetic_tp(cfg, context_for(1, "cuda"), dtype=dtype, device=torch.device("cuda"))
        _CACHE[dtype] = gpu, OracleModel(OracleConfig.of(cfg), checkpoint_tensors(cfg), tp=1), cfg
    return _CACHE[dtype]


def _log_probs(oracle, ids):
    """fp64 log-softmax of the oracle's logits after each row of ids (the whole sequence is run anew)."""
    oracle.reset(*ids.shape)
    return torch.log_softmax(oracle.forward(ids, torch.arange(ids.shape[1]))[:, -1].double(), -1)


def _plain_beam(oracle, ids, new, w, eos):
    """Beam search by the definition, every hypothesis run from its first token."""
    out = []
    for row in ids:
        hyps = [(0.0, row.tolist(), False)]
        for _ in range(new):
            cand = []
            live = [h for h in hyps if not h[2]]
            lp = _log_probs(oracle, torch.tensor([h[1] for h in live])) if live else None
            at = 0
            for b, (sc, seq, fin) in enumerate(hyps):
                if fin:
                    cand.append((sc, b, eos, seq))
                    continue
                top = lp[at].topk(w)
                at += 1
                cand += [(sc + float(v), b, int(t), seq) for v, t in zip(top.values, top.indices)]
            cand.sort(key=lambda c: (-c[0], c[1], c[2]))
            hyps = [(sc, seq + [t], t == eos) for sc, b, t, seq in cand[:w]]
        out.append(hyps)
    return out


def _prompt(cfg, b, n, seed):
    return torch.randint(0, cfg.vocab_size, (b, n), generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("b,p,new,w", [(1, 8, 12, 4), (3, 5, 6, 2), (2, 1, 5, 8), (1, 20, 1, 3), (1, 7, 9, 1)])
def test_generate_beam_fp32(lib, b, p, new, w):
    from minitp_b200.beam import generate_beam

    gpu, oracle, cfg = _models()
    ids = _prompt(cfg, b, p, b * 10 + p)
    got, scores = generate_beam(gpu, ids.cuda(), new, w, num_return=w)
    again, _ = generate_beam(gpu, ids.cuda(), new, w, num_return=w)  # the kept session's graph
    assert torch.equal(got, again)
    want = _plain_beam(oracle, ids, new, w, eos=-1)
    for i in range(b):
        assert got[i].tolist() == [h[1] for h in want[i]]
        # fp32 logits within 1e-4 of the oracle's largest: every step's log-probability within twice that
        assert scores[i].tolist() == pytest.approx([h[0] for h in want[i]], abs=2e-4 * new)
    assert gpu.ctx.comm().status() == 0


def test_generate_beam_end_token(lib):
    from minitp_b200.beam import generate_beam

    gpu, oracle, cfg = _models()
    ids = _prompt(cfg, 2, 6, 5)
    free, _ = generate_beam(gpu, ids.cuda(), 8, 4, num_return=4)
    eos = int(free[0, 1, 6 + 3])  # a token that a good hypothesis emits on its way
    got, scores = generate_beam(gpu, ids.cuda(), 8, 4, eos_token_id=eos, num_return=4, early_stop=False)
    want = _plain_beam(oracle, ids, 8, 4, eos)
    for i in range(2):
        assert got[i].tolist() == [h[1] for h in want[i]]
        assert scores[i].tolist() == pytest.approx([h[0] for h in want[i]], abs=2e-3)
    norm, ns = generate_beam(gpu, ids.cuda(), 8, 4, eos_token_id=eos, num_return=4, length_penalty=1.0)
    assert bool((ns[:, :-1] >= ns[:, 1:]).all())
    for i in range(2):
        length = [len(h[1]) - 6 if eos not in h[1][6:] else h[1][6:].index(eos) + 1 for h in want[i]]
        assert ns[i].tolist() == pytest.approx(sorted((h[0] / n for h, n in zip(want[i], length)), reverse=True), abs=2e-3)


def test_generate_beam_of_one_is_greedy(lib):
    from minitp_b200.beam import generate_beam
    from minitp_b200.generation import generate_greedy

    gpu, _, cfg = _models()
    ids = _prompt(cfg, 3, 9, 1).cuda()
    got, scores = generate_beam(gpu, ids, 20, 1)
    assert torch.equal(got[:, 0], generate_greedy(gpu, ids, 20, early_stop=False))
    assert scores.shape == (3, 1) and bool((scores < 0).all())


def test_generate_beam_stops_when_all_beams_ended(lib):
    from minitp_b200.beam import generate_beam

    gpu, _, cfg = _models()
    ids = _prompt(cfg, 1, 6, 7).cuda()
    free, _ = generate_beam(gpu, ids, 10, 1)
    eos = int(free[0, 0, 8])
    got, _ = generate_beam(gpu, ids, 10, 1, eos_token_id=eos)
    end = free[0, 0, 6:].tolist().index(eos)
    assert got.shape[2] == 6 + end + 1 and torch.equal(got[0, 0], free[0, 0, : 6 + end + 1])


def test_more_beams_than_tokens(lib):
    """A vocabulary smaller than the number of beams leaves places without a candidate in the first step."""
    from minitp_b200 import ops

    x = torch.randn(1, 1, 5, generator=torch.Generator().manual_seed(0))
    out, par, tok, _ = ops.beam_select(x.cuda(), torch.zeros(1, 1).cuda(), 8)
    assert torch.isinf(out[0, 5:]).all() and sorted(tok[0, :5].tolist()) == [0, 1, 2, 3, 4]
    # and the next step goes on from the five in use
    y = torch.randn(1, 8, 5, generator=torch.Generator().manual_seed(1))
    nxt = ops.beam_select(y.cuda(), out, 8)
    assert torch.isfinite(nxt[0]).all() and int(nxt[1].max()) < 5


@pytest.mark.parametrize("g,n,p,t,new", [(1, 3, 10, 4, 8), (2, 4, 33, 1, 5), (1, 9, 70, 20, 6)])
def test_generate_shared_prefix_equals_whole_prompts(lib, g, n, p, t, new):
    """fp32: the tokens of the same prompts run whole by the oracle."""
    from minitp_b200.beam import generate_shared_prefix

    gpu, oracle, cfg = _models()
    pre, ids = _prompt(cfg, g, p, 3), _prompt(cfg, n, t, 4)
    whole = torch.cat([pre.repeat_interleave(n // g, 0), ids], 1)
    want = oracle.generate(whole, new)[:, p:]
    for _ in range(2):
        got = generate_shared_prefix(gpu, pre.cuda(), ids.cuda(), new)
        assert torch.equal(got.cpu(), want)
    eos = int(want[0, t + 2])
    stop = generate_shared_prefix(gpu, pre.cuda(), ids.cuda(), new, eos_token_id=eos)
    for i in range(n):
        row, ref = stop[i, t:].tolist(), want[i, t:].tolist()
        end = ref.index(eos) + 1 if eos in ref else len(ref)
        assert row[:end] == ref[: len(row)][:end] and all(x == eos for x in row[end:])
    assert gpu.ctx.comm().status() == 0


def test_forward_behind_a_prefix_poisoned_caches(lib):
    """Chunked forwards behind a prefix, with NaN in every slot that holds no token."""
    from minitp_b200.generation import make_kv_cache

    gpu, oracle, cfg = _models()
    pre, ids = _prompt(cfg, 2, 37, 1), _prompt(cfg, 4, 11, 2)
    prefix, own = make_kv_cache(gpu, 2, 50), make_kv_cache(gpu, 4, 16)
    prefix.poison()
    own.poison()
    gpu(pre.cuda(), kv_cache=prefix)
    a = gpu(ids[:, :6].cuda(), kv_cache=own, prefix_cache=prefix)
    b = gpu(ids[:, 6:7].cuda(), kv_cache=own, prefix_cache=prefix)
    c = gpu(ids[:, 7:].cuda(), kv_cache=own, prefix_cache=prefix)
    got = torch.cat([a, b, c], 1).cpu()
    whole = torch.cat([pre.repeat_interleave(2, 0), ids], 1)
    full = gpu(whole.cuda()).cpu()[:, 37:]
    err = float((got - full).abs().max() / full.abs().max())
    assert err <= 1e-4 and math.isfinite(err)  # the framework's fp32 logit tolerance
    assert own.seq_len == 11


def test_forward_behind_a_prefix_in_chunks(lib):
    """More (row, token) pairs than one collective message holds go in chunks of tokens: the logits of each row are
    those of a call of a few rows."""
    from minitp_b200.generation import make_kv_cache

    gpu, _, cfg = _models()
    groups, n, t = 4, 512, 100  # 512 * 100 * 64 fp32 values, more than 8 MB
    pre, ids = _prompt(cfg, groups, 70, 1).cuda(), _prompt(cfg, n, t, 2).cuda()
    prefix, own = make_kv_cache(gpu, groups, 70), make_kv_cache(gpu, n, t + 1)
    own.poison()
    gpu(pre, kv_cache=prefix)
    got = gpu(ids, kv_cache=own, prefix_cache=prefix)
    nxt = gpu(ids[:, :1], kv_cache=own, prefix_cache=prefix)
    for g, rows in ((0, slice(0, 3)), (1, slice(250, 256)), (3, slice(509, 512))):
        one, mine = make_kv_cache(gpu, 1, 70), make_kv_cache(gpu, rows.stop - rows.start, t + 1)
        gpu(pre[g:g + 1], kv_cache=one)
        want = gpu(ids[rows], kv_cache=mine, prefix_cache=one)
        assert float((got[rows] - want).abs().max() / want.abs().max()) <= 1e-4  # the framework's fp32 logit tolerance
        want = gpu(ids[rows, :1], kv_cache=mine, prefix_cache=one)
        assert float((nxt[rows] - want).abs().max() / want.abs().max()) <= 1e-4
    assert gpu.ctx.comm().status() == 0


def test_forward_refuses_caches_that_do_not_fit(lib):
    from minitp_b200.beam import generate_beam, generate_shared_prefix
    from minitp_b200.generation import make_kv_cache

    gpu, _, cfg = _models()
    ids = _prompt(cfg, 3, 2, 1).cuda()
    prefix = make_kv_cache(gpu, 2, 8)
    gpu(ids[:2], kv_cache=prefix)
    with pytest.raises(ValueError, match="divide"):
        gpu(ids, kv_cache=make_kv_cache(gpu, 3, 8), prefix_cache=prefix)
    with pytest.raises(ValueError, match="rows"):
        gpu(ids[:2], kv_cache=make_kv_cache(gpu, 4, 8), prefix_cache=prefix)
    with pytest.raises(ValueError, match="overflow"):
        gpu(ids[:2], kv_cache=make_kv_cache(gpu, 2, 1), prefix_cache=prefix)
    for bad in (dict(num_beams=0), dict(num_beams=65), dict(num_beams=2, num_return=3),
                dict(num_beams=2, eos_token_id=cfg.vocab_size)):
        with pytest.raises(ValueError):
            generate_beam(gpu, ids, 4, **bad)
    with pytest.raises(ValueError, match="max_new_tokens"):
        generate_beam(gpu, ids, 0, 2)
    with pytest.raises(ValueError, match="divide"):
        generate_shared_prefix(gpu, ids[:2], ids, 4)


def test_positions_that_do_not_cover_the_tokens_are_refused(lib):
    from minitp_b200.generation import make_kv_cache

    gpu, _, cfg = _models()
    ids = _prompt(cfg, 2, 3, 1).cuda()
    prefix, own = make_kv_cache(gpu, 2, 8), make_kv_cache(gpu, 2, 8)
    gpu(ids, kv_cache=prefix)
    for bad in (torch.arange(2).cuda(), torch.arange(0).cuda(), torch.arange(3)):
        with pytest.raises(ValueError, match="positions"):
            gpu(ids, positions=bad, kv_cache=own, prefix_cache=prefix)
        with pytest.raises(ValueError, match="positions"):
            gpu(ids, positions=bad, kv_cache=own)
    assert own.seq_len == 0
    a = gpu(ids, positions=torch.arange(3, 6).cuda(), kv_cache=own, prefix_cache=prefix)
    own.seq_len = 0
    assert torch.equal(a, gpu(ids, kv_cache=own, prefix_cache=prefix))


def test_a_cache_behind_itself_is_refused(lib):
    from minitp_b200.generation import make_kv_cache

    gpu, _, cfg = _models()
    ids = _prompt(cfg, 2, 2, 1).cuda()
    cache = make_kv_cache(gpu, 2, 8)
    gpu(ids, kv_cache=cache)
    with pytest.raises(ValueError, match="another"):
        gpu(ids, kv_cache=cache, prefix_cache=cache)


def test_positions_behind_the_table_are_refused(lib):
    from minitp_b200.beam import generate_beam, generate_shared_prefix

    gpu, _, cfg = _models()
    top = cfg.max_position_embeddings
    ids = _prompt(cfg, 2, 3, 1).cuda()
    with pytest.raises(ValueError, match="positions"):
        generate_beam(gpu, ids, top - 1, 2)
    with pytest.raises(ValueError, match="positions"):
        generate_shared_prefix(gpu, ids[:1], ids, top - 4)
    assert generate_beam(gpu, ids, top - 2, 2)[0].shape == (2, 1, top + 1)
    assert generate_shared_prefix(gpu, ids[:1], ids, top - 5).shape == (2, top - 2)
    gpu.ctx.comm().raise_on_error()


def test_graphs_kept_over_a_larger_prompt(lib):
    """A later, larger prompt moves the model's buffers: the graphs captured before it are not replayed over the old ones."""
    from minitp_b200.beam import generate_beam, generate_shared_prefix
    from minitp_b200.generation import generate_greedy

    gpu, _, cfg = _models()
    gpu.release_native()  # the smallest buffers again
    pre, ids = _prompt(cfg, 1, 40, 1).cuda(), _prompt(cfg, 12, 3, 2).cuda()

    def small():
        return (generate_shared_prefix(gpu, pre, ids, 6), generate_beam(gpu, ids[:2], 6, 6)[0],
                generate_greedy(gpu, ids, 6, early_stop=False))  # 12 rows: a graph of the kernel chain

    want = small()
    for length in (100, 300):
        generate_greedy(gpu, _prompt(cfg, 14, length, 3).cuda(), 3, early_stop=False)
        generate_shared_prefix(gpu, _prompt(cfg, 1, 10 * length, 4).cuda(), ids, 3)
        torch.cuda.synchronize()
        again = small()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(again, want))
    assert gpu.ctx.comm().status() == 0


def test_greedy_sessions_stay_over_other_searches(lib):
    """Beam and shared-prefix shapes take no place of a greedy session: its buffers and graph are there for the next
    call, and all of them go with the native model."""
    from minitp_b200.beam import generate_beam, generate_shared_prefix
    from minitp_b200.generation import decode_session, generate_greedy

    gpu, _, cfg = _models()
    ids = _prompt(cfg, 2, 5, 1).cuda()
    want = generate_greedy(gpu, ids, 6, early_stop=False)
    kept = decode_session(gpu, 2, 11, ids.device)
    graph = kept.graph
    for w in range(1, 5):
        generate_beam(gpu, ids, 3, w)
        generate_beam(gpu, ids, 3, w, eos_token_id=w)
        generate_shared_prefix(gpu, ids[:1], ids[:, :w], 3)
    again = decode_session(gpu, 2, 11, ids.device)
    assert again is kept and again.graph is graph
    assert torch.equal(generate_greedy(gpu, ids, 6, early_stop=False), want)
    beams = generate_beam(gpu, ids, 3, 2)
    for n in range(1, 6):  # nor the other way round
        generate_greedy(gpu, ids, n, early_stop=False)
    assert all(torch.equal(a, b) for a, b in zip(generate_beam(gpu, ids, 3, 2), beams))
    gpu.release_native()
    assert not any(k.endswith("_sessions") for k in vars(gpu))
    assert torch.equal(generate_greedy(gpu, ids, 6, early_stop=False), want)


def test_bf16_logits_behind_a_prefix(lib):
    """bf16, the 0.5B shape with two layers: rows behind a shared prefix against the whole prompts, many tokens and
    one at a time, within the framework's bf16 logit tolerance (0.5 absolute)."""
    from minitp_b200.distributed.context import context_for
    from minitp_b200.generation import make_kv_cache
    from minitp_b200.weight_loader import load_synthetic_tp

    cfg = mcfg.qwen25_05b(num_layers=2)
    gpu = load_synthetic_tp(cfg, context_for(1, "cuda"), dtype=torch.bfloat16, device=torch.device("cuda"))
    for groups, rows, p, t, cap in ((1, 12, 1500, 40, 64), (2, 4, 200, 1, 8)):
        pre, ids = _prompt(cfg, groups, p, 1).cuda(), _prompt(cfg, rows, t + 3, 2).cuda()
        prefix, own = make_kv_cache(gpu, groups, p + 5), make_kv_cache(gpu, rows, cap)
        prefix.poison()
        own.poison()
        gpu(pre, kv_cache=prefix, last_only=True)
        got = [gpu(ids[:, :t], kv_cache=own, prefix_cache=prefix)]
        got += [gpu(ids[:, t + i:t + i + 1], kv_cache=own, prefix_cache=prefix) for i in range(3)]
        got = torch.cat(got, 1).float()
        whole = gpu(torch.cat([pre.repeat_interleave(rows // groups, 0), ids], 1))[:, p:].float()
        assert bool(torch.isfinite(got).all())
        assert float((got - whole).abs().max()) <= 0.5
        assert float((got - whole).abs().max() / whole.abs().max()) <= 0.1
    assert gpu.ctx.comm().status() == 0
