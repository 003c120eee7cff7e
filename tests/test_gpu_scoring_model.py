"""Scoring of prompts through the model: packed forwards against the oracle and against forwards of one prompt."""

import dataclasses

import pytest
import torch

from minitp_b200 import config as mcfg
from oracle.model import OracleConfig, OracleModel, checkpoint_tensors

pytestmark = pytest.mark.gpu

_CACHE: dict = {}


def _model(name, dtype=torch.float32):
    """A model of one rank on the GPU: the tiny one, or shapes with the head dims of the others."""
    if (name, dtype) not in _CACHE:
        from minitp_b200.distributed.context import context_for
        from minitp_b200.weight_loader import load_synthetic_tp

        cfg = {"tiny": mcfg.baseline_tiny(),
               "q05b": dataclasses.replace(mcfg.qwen25_05b(2), vocab_size=5003, intermediate_size=640),
               "hd128": dataclasses.replace(mcfg.qwen25_7b(2), hidden_size=768, num_attention_heads=6, num_key_value_heads=2,
                                            vocab_size=5003, intermediate_size=640)}[name]
        _CACHE[name, dtype] = load_synthetic_tp(cfg, context_for(1, "cuda"), dtype=dtype, device=torch.device("cuda")), cfg
    return _CACHE[name, dtype]


def _prompts(cfg, lengths, seed):
    r = torch.Generator().manual_seed(seed)
    return [torch.randint(0, cfg.vocab_size, (n,), generator=r) for n in lengths]


def _check(got, logits, ids, top, off):
    """`got` is the scores of `ids` by logits [n, V] that are right to within `off`: a log-probability is then off
    by twice that, and the entropy by that times (1 + H)."""
    lp = torch.log_softmax(logits.detach().cpu().double(), -1)[:-1]
    want = lp.gather(1, ids[1:, None])[:, 0]
    ent = -(lp.exp() * lp).sum(-1)
    assert got.logprobs.shape == got.entropy.shape == want.shape
    assert float((got.logprobs.cpu().double() - want).abs().max()) <= 2 * off
    assert float(((got.entropy.cpu().double() - ent).abs() / (1 + ent)).max()) <= 2 * off
    if not top:
        assert got.top_logprobs is None and got.top_ids is None
        return
    best = lp.topk(top, dim=-1).values
    assert float((got.top_logprobs.cpu().double() - best).abs().max()) <= 2 * off
    assert float((lp.gather(1, got.top_ids.cpu()) - best).abs().max()) <= 4 * off
    assert all(len(set(row)) == top for row in got.top_ids.tolist())


def test_scores_against_the_oracle_fp32(lib):
    """Prompts of all sizes, empty ones and single tokens among them, as tensors on either device and as lists."""
    from minitp_b200.scoring import score_prompts

    model, cfg = _model("tiny")
    oracle = OracleModel(OracleConfig.of(cfg), checkpoint_tensors(cfg), tp=1)
    prompts = _prompts(cfg, [7, 1, 0, 64, 2, 33, 130], 1)
    given = [prompts[0].tolist(), prompts[1], prompts[2], prompts[3].cuda(), prompts[4].int(), prompts[5], prompts[6]]
    for top, most in ((0, 32768), (5, 32768), (5, 40), (3, 1)):
        got = score_prompts(model, given, top, max_tokens=most)
        assert len(got) == len(prompts)
        for g, ids in zip(got, prompts):
            if ids.numel() < 2:
                assert g.logprobs.numel() == g.entropy.numel() == 0
                assert g.top_ids is None if top == 0 else g.top_ids.shape == (0, top)
                continue
            oracle.reset(1, ids.numel())
            logits = oracle.forward(ids[None], torch.arange(ids.numel()))[0]
            _check(g, logits, ids, top, 1e-4 * float(logits.abs().max()))  # the framework's fp32 logit tolerance
    assert model.ctx.comm().status() == 0


@pytest.mark.parametrize("name", ["q05b", "hd128"])
def test_packed_forward_is_each_prompts_own_fp32(lib, name):
    model, cfg = _model(name)
    lengths = [90, 1, 3, 257, 64, 0, 20]
    prompts = _prompts(cfg, lengths, 2)
    starts = torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32)
    hidden = model.forward_packed(torch.cat(prompts).cuda(), starts.cuda())
    logits = model.lm_head(hidden)
    for a, ids in zip(starts.tolist(), prompts):
        if ids.numel():
            want = model(ids[None].cuda())[0]
            assert float((logits[a:a + ids.numel()] - want).abs().max() / want.abs().max()) <= 1e-4
    assert model.ctx.comm().status() == 0


@pytest.mark.parametrize("name", ["q05b", "hd128"])
def test_scores_bf16(lib, name):
    from minitp_b200.scoring import score_prompts

    model, cfg = _model(name, torch.bfloat16)
    prompts = _prompts(cfg, [300, 5, 77, 128, 1, 611], 3)
    got = score_prompts(model, prompts, 4)
    for g, ids in zip(got, prompts):
        if ids.numel() > 1:
            _check(g, model(ids[None].cuda())[0], ids, 4, 0.5)  # the framework's bf16 logit tolerance
            want = torch.log_softmax(model(ids[None].cuda())[0].double(), -1)[:-1].gather(1, ids[1:, None].cuda())[:, 0]
            # two roundings of the same network: far nearer to each other than another prompt's tokens would be
            assert float((g.logprobs - want).abs().mean()) <= 0.5 * float((want - want.roll(1)).abs().mean())
    assert model.ctx.comm().status() == 0


def test_packed_forward_in_chunks(lib):
    """More tokens than one collective message holds go in chunks, cut inside a prompt: the scores are each prompt's own."""
    from minitp_b200.scoring import score_prompts

    model, cfg = _model("tiny")
    lengths = [211 + 37 * (i % 7) for i in range(120)]  # 38580 tokens of 64 fp32 values, more than 8 MB
    prompts = _prompts(cfg, lengths, 4)
    got = score_prompts(model, prompts, 2, max_tokens=1 << 20)
    at = torch.tensor(lengths).cumsum(0)
    edge = int((at <= 32768).sum())  # the prompt that the first chunk's end cuts
    for i in (0, 1, edge - 1, edge, edge + 1, 119):
        logits = model(prompts[i][None].cuda())[0]
        _check(got[i], logits, prompts[i], 2, 1e-4 * float(logits.abs().max()))
    assert model.ctx.comm().status() == 0


@pytest.mark.parametrize("name,dtype", [("tiny", torch.float32), ("q05b", torch.bfloat16)])
def test_packed_forward_of_one_token(lib, name, dtype):
    """A single token, and a last chunk of one token."""
    model, cfg = _model(name, dtype)
    ids = _prompts(cfg, [1], 10)[0].cuda()
    one = torch.tensor([0, 1], dtype=torch.int32).cuda()
    want = model(ids[None])[0]
    got = model.lm_head(model.forward_packed(ids, one))
    off = 1e-4 * float(want.abs().max()) if dtype == torch.float32 else 0.5
    assert float((got - want).abs().max()) <= off
    n = model.ctx.comm().slot_bytes() // (cfg.hidden_size * ids.new_empty(0, dtype=dtype).element_size()) + 1
    ids = _prompts(cfg, [n], 11)[0].cuda()
    starts = torch.tensor([*range(0, n - 40, 1000), n - 40, n], dtype=torch.int32).cuda()
    got = model.lm_head(model.forward_packed(ids, starts)[n - 40:])
    want = model(ids[None, n - 40:])[0]
    assert float((got - want).abs().max()) <= (1e-4 * float(want.abs().max()) if dtype == torch.float32 else 0.5)
    assert model.ctx.comm().status() == 0


def test_prompts_longer_than_the_position_table_are_flagged(lib):
    model, cfg = _model("tiny")
    ids = _prompts(cfg, [cfg.max_position_embeddings + 9], 12)[0].cuda()
    model.forward_packed(ids, torch.tensor([0, 8, ids.numel() - 1], dtype=torch.int32).cuda())
    assert model.ctx.comm().status() == 0
    model.forward_packed(ids, torch.tensor([0, ids.numel()], dtype=torch.int32).cuda())
    assert model.ctx.comm().status() == 2
    model.ctx.comm().clear_status()


def test_tokens_of_no_prompt_change_nothing(lib):
    model, cfg = _model("tiny")
    ids = _prompts(cfg, [100], 5)[0].cuda()
    a = model.forward_packed(ids, torch.tensor([10, 40, 90], dtype=torch.int32).cuda())
    other = ids.clone()
    other[:10], other[90:] = 3, 4
    b = model.forward_packed(other, torch.tensor([10, 40, 90], dtype=torch.int32).cuda())
    assert torch.equal(a[10:90], b[10:90]) and bool(torch.isfinite(a).all())
    want = model(ids[None, 40:90])[0]
    got = model.lm_head(a[40:90])
    assert float((got - want).abs().max() / want.abs().max()) <= 1e-4


def test_given_positions(lib):
    model, cfg = _model("tiny")
    ids = _prompts(cfg, [60], 6)[0].cuda()
    st = torch.tensor([0, 25, 60], dtype=torch.int32).cuda()
    pos = torch.cat([torch.arange(25), torch.arange(35)]).cuda()
    assert torch.equal(model.forward_packed(ids, st), model.forward_packed(ids, st, pos))
    want = model(ids[None, 25:], positions=torch.arange(7, 42).cuda())[0]
    got = model.lm_head(model.forward_packed(ids, st, torch.cat([torch.arange(25), torch.arange(7, 42)]).cuda())[25:])
    assert float((got - want).abs().max() / want.abs().max()) <= 1e-4


def test_packed_forward_captured(lib):
    """A captured forward replays on other tokens and other prompts."""
    model, cfg = _model("q05b", torch.bfloat16)
    ids, other = _prompts(cfg, [200, 200], 7)
    x, st = ids.cuda(), torch.tensor([0, 50, 200], dtype=torch.int32).cuda()
    model.forward_packed(x, st)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = model.forward_packed(x, st)
    x.copy_(other), st.copy_(torch.tensor([0, 120, 180], dtype=torch.int32))
    g.replay()
    want = model.forward_packed(other.cuda(), torch.tensor([0, 120, 180], dtype=torch.int32).cuda())
    assert torch.equal(out, want)


def test_greedy_generation_around_scoring(lib):
    """Sessions kept by greedy decoding stay right when a scoring call has moved the model's buffers."""
    from minitp_b200.generation import generate_greedy
    from minitp_b200.scoring import score_prompts

    cfg = mcfg.baseline_tiny()
    from minitp_b200.distributed.context import context_for
    from minitp_b200.weight_loader import load_synthetic_tp

    model = load_synthetic_tp(cfg, context_for(1, "cuda"), dtype=torch.float32, device=torch.device("cuda"))
    ids = torch.stack(_prompts(cfg, [12] * 10, 8)).cuda()
    first = generate_greedy(model, ids, 9, early_stop=False)
    score_prompts(model, _prompts(cfg, [400, 500, 600], 9))
    assert torch.equal(generate_greedy(model, ids, 9, early_stop=False), first)


def test_many_empty_prompts(lib):
    """Prompts of no token add none to a forward, however many there are."""
    from minitp_b200.scoring import score_prompts

    model, cfg = _model("tiny")
    ids = _prompts(cfg, [7, 5], 10)
    want = score_prompts(model, ids, 2)
    none = ids[0][:0]
    got = score_prompts(model, [ids[0], *[none] * 70000, ids[1]], 2)
    assert len(got) == 70002 and all(g.logprobs.numel() == 0 for g in got[1:-1])
    for g, w in zip((got[0], got[-1]), want):
        assert torch.allclose(g.logprobs, w.logprobs, rtol=0, atol=1e-4) and g.top_ids.shape == w.top_ids.shape


def test_scoring_refusals(lib):
    from minitp_b200.scoring import score_prompts

    model, cfg = _model("tiny")
    for prompts, kw, match in [([[1, 2]], dict(top=65), "top"), ([[1, 2]], dict(max_tokens=0), "max_tokens"),
                               ([torch.zeros(2, 2, dtype=torch.int64)], {}, "sequences"), ([torch.zeros(3)], {}, "sequences"),
                               ([[0, cfg.vocab_size]], {}, "vocabulary"), ([[0, -1]], {}, "vocabulary"),
                               ([torch.zeros(cfg.max_position_embeddings + 1, dtype=torch.int64)], {}, "positions")]:
        with pytest.raises(ValueError, match=match):
            score_prompts(model, prompts, **kw)
    ids, st = torch.zeros(4, dtype=torch.int64).cuda(), torch.tensor([0, 4], dtype=torch.int32).cuda()
    for args, match in [((ids[None], st), "input_ids"), ((ids[:0], st), "input_ids"), ((ids, st.long()), "seq_starts"),
                        ((ids, st, torch.zeros(3, dtype=torch.int64).cuda()), "positions")]:
        with pytest.raises(ValueError, match=match):
            model.forward_packed(*args)
    assert score_prompts(model, []) == []
