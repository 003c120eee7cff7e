"""Packed prompt attention and token log-probabilities against plain 64-bit implementations."""

import math

import pytest
import torch

from tests import scoring_ref

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _starts(lengths, at=0):
    out = [at]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _cuda_starts(starts):
    return torch.tensor(starts, dtype=torch.int32, device="cuda")


def _parts(r, total, hq, hkv, hd, dtype):
    """q, k and v as parts of one projection's output, on the GPU."""
    qkv = torch.randn(total, hq + 2 * hkv, hd, generator=r).to(DT[dtype]).cuda()
    return qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]


def _close(got, want, tol):
    got = got.detach().cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN elsewhere"
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    off = (got - want).abs()[fine] - tol[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, float(off.max())


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("hq,hkv,hd", [(4, 2, 16), (8, 4, 32), (14, 2, 64), (3, 3, 64), (7, 1, 128), (16, 2, 128)])
@pytest.mark.parametrize("lengths", [[1], [0, 5, 0], [128], [129, 127, 1, 300], [17, 64, 33], [401]])
def test_prompt_attention(lib, dtype, hq, hkv, hd, lengths):
    from minitp_b200 import ops

    starts = _starts(lengths)
    q, k, v = _parts(_gen(hq + hd + sum(lengths)), starts[-1], hq, hkv, hd, dtype)
    got = ops.prompt_attention(q, k, v, _cuda_starts(starts))
    assert got.dtype == q.dtype and got.is_contiguous()
    _close(got, *scoring_ref.attend(q, k, v, starts))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("hq,hkv,hd", [(4, 2, 16), (14, 2, 64), (4, 1, 128)])
def test_prompt_attention_many_prompts(lib, dtype, hq, hkv, hd):
    """More prompts than are put in order (127, 128, 129, 300), empty ones among them."""
    from minitp_b200 import ops

    for count in (127, 128, 129, 300):
        r = _gen(count)
        lengths = torch.randint(0, 9, (count,), generator=r).tolist()
        lengths[count // 2] = 90
        starts = _starts(lengths)
        q, k, v = _parts(r, starts[-1], hq, hkv, hd, dtype)
        _close(ops.prompt_attention(q, k, v, _cuda_starts(starts)), *scoring_ref.attend(q, k, v, starts))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("hq,hkv,hd", [(40, 1, 64), (130, 1, 64), (300, 1, 128), (131, 1, 64), (257, 1, 16)])
def test_prompt_attention_many_heads_a_kv_head(lib, dtype, hq, hkv, hd):
    """More query heads of a KV head than a tile has rows, prime numbers of them too."""
    from minitp_b200 import ops

    starts = _starts([19, 1, 40])
    q, k, v = _parts(_gen(hq), starts[-1], hq, hkv, hd, dtype)
    _close(ops.prompt_attention(q, k, v, _cuda_starts(starts)), *scoring_ref.attend(q, k, v, starts))


@pytest.mark.parametrize("dtype,hq,hkv,hd", [("fp32", 4, 2, 16), ("bf16", 14, 2, 64), ("bf16", 4, 4, 128)])
def test_prompt_attention_thousands_of_prompts(lib, dtype, hq, hkv, hd):
    from minitp_b200 import ops

    lengths = torch.randint(0, 13, (5000,), generator=_gen(1)).tolist()
    starts = _starts(lengths, at=3)
    q, k, v = _parts(_gen(2), starts[-1] + 5, hq, hkv, hd, dtype)
    got = ops.prompt_attention(q, k, v, _cuda_starts(starts))
    want, tol = scoring_ref.attend(q, k, v, starts)
    _close(got, want, tol)
    part = ops.prompt_attention(q[1000:9001], k, v, _cuda_starts(starts), first=1000)
    _close(part, want[1000:9001], tol[1000:9001])


def test_two_calls_at_once(lib):
    """Calls of every kind on two streams at the same time: each call's results are its own."""
    from minitp_b200 import ops

    streams = [torch.cuda.Stream() for _ in range(2)]
    q, k, v = _parts(_gen(50), 3000, 14, 2, 64, "bf16")
    starts = [_cuda_starts([0, 1700, 3000]), _cuda_starts([0, 40, 2000, 3000])]
    x = torch.randn(600, 30000, generator=_gen(51)).cuda()
    t = torch.randint(0, 30000, (600,), generator=_gen(52)).cuda()
    alone = [(ops.prompt_attention(q, k, v, s), *ops.token_logprobs(x[i * 50:], t[i * 50:], 7 - i)) for i, s in enumerate(starts)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for i, (st, s) in enumerate(zip(streams, starts)):
            with torch.cuda.stream(st):
                got.append((ops.prompt_attention(q, k, v, s), *ops.token_logprobs(x[i * 50:], t[i * 50:], 7 - i)))
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            for y, z in zip(a, b):
                assert torch.equal(y, z)


@pytest.mark.parametrize("dtype,hq,hkv,hd", [("fp32", 4, 2, 16), ("bf16", 14, 2, 64), ("bf16", 8, 2, 128), ("bf16", 6, 3, 32)])
def test_prompt_attention_pieces(lib, dtype, hq, hkv, hd):
    """Queries of a piece of the packed tokens give the whole call's rows, wherever the pieces are cut."""
    from minitp_b200 import ops

    starts = _starts([40, 1, 0, 300, 77])
    q, k, v = _parts(_gen(3), starts[-1], hq, hkv, hd, dtype)
    want, tol = scoring_ref.attend(q, k, v, starts)
    for cuts in ([0, 418], [0, 7, 40, 41, 200, 418], [0, 417, 418], [100, 101, 355]):
        for a, b in zip(cuts, cuts[1:]):
            _close(ops.prompt_attention(q[a:b], k, v, _cuda_starts(starts), first=a), want[a:b], tol[a:b])


@pytest.mark.parametrize("dtype,hq,hkv,hd", [("fp32", 4, 2, 16), ("bf16", 14, 2, 64), ("bf16", 4, 1, 128)])
def test_prompt_attention_tokens_of_no_prompt_get_zero(lib, dtype, hq, hkv, hd):
    """Rows before the first and behind the last prompt become 0, and what they hold reaches nothing."""
    from minitp_b200 import ops

    total = 500
    q, k, v = _parts(_gen(9), total, hq, hkv, hd, dtype)
    for starts in ([13, 50, 50, 301], [0, 3], [499, 500], [7], [500, 500], [0, 500], [250, 250, 250]):
        q2, k2, v2 = q.clone(), k.clone(), v.clone()
        for t in (q2, k2, v2):
            t[:starts[0]] = math.nan
            t[starts[-1]:] = math.nan
        got = ops.prompt_attention(q2, k2, v2, _cuda_starts(starts))
        assert not got[:starts[0]].any() and not got[starts[-1]:].any()
        want, tol = scoring_ref.attend(q, k, v, starts)
        _close(got[starts[0]:starts[-1]], want[starts[0]:starts[-1]], tol[starts[0]:starts[-1]])
        part = ops.prompt_attention(q2[5:490], k2, v2, _cuda_starts(starts), first=5)
        a, b = max(5, starts[0]), min(490, starts[-1])
        assert not part[:max(0, a - 5)].any() and not part[max(0, b - 5):].any()
        if b > a:
            _close(part[a - 5:b - 5], want[a:b], tol[a:b])


@pytest.mark.parametrize("dtype,hq,hkv,hd", [("fp32", 4, 2, 16), ("bf16", 14, 2, 64), ("bf16", 4, 1, 128)])
def test_prompt_attention_starts_out_of_range(lib, dtype, hq, hkv, hd):
    """Starts that decrease or lie outside the tokens are cut to what fits: no access leaves the tensors."""
    from minitp_b200 import ops

    q, k, v = _parts(_gen(4), 200, hq, hkv, hd, dtype)
    for given, meant in [([-5, 20, 900], [0, 20, 200]), ([50, 30, 120], [50, 50, 120]), ([300, 400], [200, 200]),
                         ([-(2 ** 31), 2 ** 31 - 1], [0, 200])]:
        got = ops.prompt_attention(q, k, v, _cuda_starts(given))
        want, tol = scoring_ref.attend(q, k, v, meant)
        _close(got, want, tol)


@pytest.mark.parametrize("dtype,hq,hkv,hd", [("fp32", 4, 2, 16), ("fp32", 2, 1, 128), ("bf16", 14, 2, 64), ("bf16", 4, 1, 128)])
def test_prompt_attention_nan_and_infinities(lib, dtype, hq, hkv, hd):
    """A NaN or an infinity of K or V reaches the tokens that see it, and no other prompt or earlier token."""
    from minitp_b200 import ops

    starts = _starts([150, 40, 200])
    q, k, v = (t.clone() for t in _parts(_gen(5), starts[-1], hq, hkv, hd, dtype))
    v[100, 0, 3] = math.nan
    v[149, 0, 5] = math.inf
    v[189, hkv - 1, 7] = -math.inf
    k[190 + 130, 0, 2] = math.nan  # later tokens' scores
    v[190 + 199, 0, 1] = math.nan  # the last token alone
    got = ops.prompt_attention(q, k, v, _cuda_starts(starts))
    want, tol = scoring_ref.attend(q, k, v, starts)
    per = hq // hkv
    seen = want.clone()
    seen[190 + 130:, :per] = math.nan  # a NaN score makes its row NaN
    _close(got, seen, tol)


@pytest.mark.parametrize("dtype,hd", [("fp32", 16), ("bf16", 64), ("bf16", 128)])
def test_prompt_attention_scores_of_minus_infinity(lib, dtype, hd):
    """Keys whose scores are -inf count for nothing; a token that sees no other gets 0."""
    from minitp_b200 import ops

    starts = _starts([30, 170])
    q, k, v = (t.clone() for t in _parts(_gen(6), starts[-1], 4, 2, hd, dtype))
    q[..., 0] = 1.0
    for j in (30, 31, 32, 60, 199):
        k[j, :, 0] = -math.inf
    got = ops.prompt_attention(q, k, v, _cuda_starts(starts))
    assert not got[30:33].any()
    _close(got, *scoring_ref.attend(q, k, v, starts))


@pytest.mark.parametrize("dtype,hd", [("fp32", 32), ("bf16", 64), ("bf16", 128)])
def test_prompt_attention_large_scores(lib, dtype, hd):
    """Scores of some thousands, growing along the prompt (the running maximum moves at every tile) or falling."""
    from minitp_b200 import ops

    n, starts = 600, _starts([600])
    q, k, v = (t.clone() for t in _parts(_gen(7), n, 4, 2, hd, dtype))
    q[..., 0] = 40.0
    for sign in (1, -1):
        k[..., 0] = (sign * torch.arange(n) * 0.5).to(k.dtype).cuda()[:, None]
        _close(ops.prompt_attention(q, k, v, _cuda_starts(starts)), *scoring_ref.attend(q, k, v, starts))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("hd", [16, 64, 128])
def test_prompt_attention_strides(lib, dtype, hd):
    """Contiguous tensors, heads before tokens (a cache's layout), padded rows, a gap between heads, an unaligned
    view and an expanded head: one result."""
    from minitp_b200 import ops

    starts = _starts([70, 1, 130])
    n = starts[-1]
    r = _gen(8)
    q = torch.randn(n, 6, hd, generator=r).to(DT[dtype]).cuda()
    k, v = (torch.randn(n, 2, hd, generator=r).to(DT[dtype]).cuda() for _ in range(2))
    st = _cuda_starts(starts)
    want = ops.prompt_attention(q, k, v, st)
    _close(want, *scoring_ref.attend(q, k, v, starts))

    def heads_first(t):
        return t.transpose(0, 1).contiguous().transpose(0, 1)

    def padded(t):
        w = torch.full((t.shape[0] + 3, t.shape[1] + 2, hd + 16), math.nan, dtype=t.dtype, device="cuda")
        w[1:n + 1, 1:t.shape[1] + 1, 16:] = t
        return w[1:n + 1, 1:t.shape[1] + 1, 16:]

    def unaligned(t):
        w = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        w[1:] = t.reshape(-1)
        return w[1:].view(t.shape)

    def dims_strided(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    for f in (heads_first, padded, unaligned, dims_strided):
        assert torch.equal(ops.prompt_attention(f(q), f(k), f(v), st), want)
    k1, v1 = k[:, :1].contiguous().expand(n, 2, hd), v[:, :1].contiguous().expand(n, 2, hd)
    assert torch.equal(ops.prompt_attention(q, k1, v1, st), ops.prompt_attention(q, k1.contiguous(), v1.contiguous(), st))


@pytest.mark.parametrize("dtype,heads_apart", [("bf16", False), ("fp32", False), ("bf16", True), ("fp32", True)])
def test_prompt_attention_offsets_past_32_bits(lib, dtype, heads_apart):
    """Tokens, or heads, that lie more than 2^31 elements apart."""
    from minitp_b200 import ops

    starts = [0, 3, 5]
    far = 2 ** 29 + 64 if not heads_apart else 2 ** 28 + 64  # 5 tokens, or 8 heads
    r = _gen(15)
    packed = torch.randn(5, 8, 64, generator=r).to(DT[dtype]).cuda()
    buf = torch.empty(4 * far + 8 * 64 if not heads_apart else 7 * far + 5 * 64, dtype=DT[dtype], device="cuda")
    wide = buf.as_strided((5, 8, 64), (64, far, 1) if heads_apart else (far, 64, 1))
    wide.copy_(packed)
    (q, k, v), (fq, fk, fv) = ((t[:, :4], t[:, 4:6], t[:, 6:]) for t in (packed, wide))
    if heads_apart:  # (two heads are not far apart: the second KV head is the last but one)
        fk, fv, k, v = wide[:, 0:8:7], wide[:, 1:8:6], packed[:, 0:8:7], packed[:, 1:8:6]
    st = _cuda_starts(starts)
    got = ops.prompt_attention(fq, fk, fv, st)
    _close(got, *scoring_ref.attend(q, k, v, starts))
    assert torch.equal(got, ops.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), st))


def test_prompt_attention_empty(lib):
    from minitp_b200 import ops

    q, k = torch.zeros(0, 4, 64, device="cuda"), torch.zeros(0, 2, 64, device="cuda")
    assert ops.prompt_attention(q, k, k, _cuda_starts([0, 0])).shape == (0, 4, 64)


def test_prompt_attention_refusals(lib):
    from minitp_b200 import _lib, ops

    q, k = torch.zeros(5, 4, 64, device="cuda"), torch.zeros(5, 2, 64, device="cuda")
    st = _cuda_starts([0, 5])
    for args, match in [((q, k, k[:, :1], st), "need q"), ((q[0], k, k, st), "need q"), ((q, k.bfloat16(), k, st), "dtype"),
                        ((q, k, k, st.long()), "int32"), ((q, k, k, st[:0]), "int32"), ((q[:, :3], k, k, st), "heads"),
                        ((q.half(), k.half(), k.half(), st), "unsupported dtype"), ((q, k, k, st, 1), "tokens"),
                        ((q[..., :40].contiguous(), k[..., :40].contiguous(), k[..., :40].contiguous(), st), "head_dim"),
                        ((q, k, k, st.cpu()), "CUDA")]:
        with pytest.raises(_lib.MinitpB200Error, match=match):
            ops.prompt_attention(*args)


def test_prompt_attention_captured_and_on_another_stream(lib):
    """A captured call replays on new contents and new starts; another stream's call gives the same."""
    from minitp_b200 import ops

    for dtype, hq, hkv, hd in [("fp32", 4, 2, 16), ("bf16", 14, 2, 64), ("bf16", 4, 1, 128)]:
        q, k, v = _parts(_gen(10), 300, hq, hkv, hd, dtype)
        st = _cuda_starts([0, 200, 300])
        ops.prompt_attention(q, k, v, st)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.prompt_attention(q, k, v, st)
        side = torch.cuda.Stream()
        for seed, starts in [(11, [0, 1, 300]), (12, [20, 150, 299])]:
            nq, nk, nv = _parts(_gen(seed), 300, hq, hkv, hd, dtype)
            q.copy_(nq), k.copy_(nk), v.copy_(nv), st.copy_(_cuda_starts(starts))
            g.replay()
            _close(out, *scoring_ref.attend(nq, nk, nv, starts))
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                other = ops.prompt_attention(q, k, v, st)
            side.synchronize()
            assert torch.equal(other, out)


@pytest.mark.parametrize("dtype,hq,hkv,hd", [("bf16", 14, 2, 64), ("bf16", 8, 2, 128)])
def test_prompt_attention_long_prompt(lib, dtype, hq, hkv, hd):
    """A few thousand tokens beside short prompts; the rows that see the most and the fewest keys."""
    from minitp_b200 import ops

    starts = _starts([3001, 100, 2500])
    q, k, v = _parts(_gen(13), starts[-1], hq, hkv, hd, dtype)
    got = ops.prompt_attention(q, k, v, _cuda_starts(starts))
    for a, b in [(0, 64), (2950, 3001), (3001, 3101), (5500, 5601)]:
        want, tol = scoring_ref.attend(q[a:b], k, v, starts, first=a)
        _close(got[a:b], want, tol)


@pytest.mark.parametrize("dtype,hd", [("fp32", 16), ("fp32", 32), ("fp32", 64), ("fp32", 128), ("bf16", 16), ("bf16", 32)])
@pytest.mark.parametrize("lengths", [[40, 1, 61], [150, 0, 1, 201], [700, 1, 0, 450, 31]])
def test_prompt_attention_row_tiles_of_every_size(lib, dtype, hd, lengths):
    """Few, more and many rows, which take tiles of 16, 32 and 64 rows on the CUDA cores; values that are not finite."""
    from minitp_b200 import ops

    starts = _starts(lengths, at=2)
    q, k, v = (t.clone() for t in _parts(_gen(17 + hd), starts[-1] + 3, 20, 4, hd, dtype))
    v[starts[1] - 1, 0, 3] = math.nan  # the first prompt's last token alone
    v[starts[-2] + 20, 1, 5] = math.inf
    v[starts[-1] - 1, 3, 7] = -math.inf
    got = ops.prompt_attention(q, k, v, _cuda_starts(starts))
    _close(got, *scoring_ref.attend(q, k, v, starts))
    a, b = starts[1] - 5, starts[-1] + 1  # a piece that begins and ends inside a tile
    want, tol = scoring_ref.attend(q[a:b], k, v, starts, first=a)
    _close(ops.prompt_attention(q[a:b], k, v, _cuda_starts(starts), first=a), want, tol)


# ------------------------------------------------------------------ log-probabilities
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,v,top", [(1, 1, 1), (1, 1000, 4), (3, 7, 7), (2, 7, 20), (5, 4097, 0), (4, 151936, 5),
                                        (2, 151937, 64), (40, 20001, 20), (300, 333, 64), (700, 2048, 1), (9, 8192, 33)])
def test_token_logprobs(lib, dtype, rows, v, top):
    from minitp_b200 import ops

    r = _gen(rows + v + top)
    x = (torch.randn(rows, v, generator=r) * 3).to(DT[dtype])
    t = torch.randint(0, v, (rows,), generator=r)
    t[::2] = x[::2].argmax(-1)
    scoring_ref.check_logprobs(ops.token_logprobs(x.cuda(), t.cuda(), top), x, t, top)
    scoring_ref.check_logprobs(ops.token_logprobs(x.cuda(), None, top), x, None, top)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_token_logprobs_ties_go_to_the_lowest_id(lib, dtype):
    from minitp_b200 import ops

    for v, top in [(20, 6), (9000, 16), (30000, 64)]:
        x = torch.zeros(3, v, dtype=DT[dtype])
        x[0, 5] = -0.0  # the same value as +0.0
        x[1] = torch.randint(0, 3, (v,), generator=_gen(v)).to(DT[dtype])
        x[2] = torch.randint(-2, 1, (v,), generator=_gen(v + 1)).to(DT[dtype]) * 20
        t = torch.tensor([5, v - 1, 0])
        scoring_ref.check_logprobs(ops.token_logprobs(x.cuda(), t.cuda(), top), x, t, top)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("v", [40, 20000])
def test_token_logprobs_masks_infinities_and_nan(lib, dtype, v):
    from minitp_b200 import ops

    inf, nan = math.inf, math.nan
    low = torch.finfo(DT[dtype]).min
    x = torch.full((9, v), -inf)
    x[0, :3] = torch.tensor([1.0, nan, 2.0])
    x[1, v - 1] = 0.5  # one token left
    x[3, 4:6] = inf  # shared by two
    x[3, 8] = 3.0
    x[4] = low  # masked by the type's lowest value: a uniform row
    x[5] = nan
    x[6] = torch.randn(v, generator=_gen(1))
    x[6, ::3] = low
    x[7] = torch.randn(v, generator=_gen(2))
    x[7, 1::2] = -inf
    x[8, 7] = low
    x[8, 9] = torch.finfo(DT[dtype]).max
    x = x.to(DT[dtype])
    for t in ([0, v - 1, 3, 4, 9, 1, 3, 2, 7], [1, 0, 0, 8, v - 1, 2, 4, 1, 9], [-1, v, v + 5, -100, 2 ** 40, -2 ** 40, 0, 0, 8]):
        for top in (0, 1, 5, 50):
            tt = torch.tensor(t)
            scoring_ref.check_logprobs(ops.token_logprobs(x.cuda(), tt.cuda(), top), x, tt, top)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("v", [333, 20001])
def test_token_logprobs_logits_of_every_size(lib, dtype, v):
    """Rows far from zero, of every spread, and around 2^30 and 2^38, where neighbours lie far apart."""
    from minitp_b200 import ops

    r = _gen(v)
    rows = [torch.randn(v, generator=r) * 3 + d for d in (-1e4, 1e4, -1e6, 1e6, 3e7, -3e8, 1e9, -1e12)]
    rows += [torch.randn(v, generator=r) * 10.0 ** e for e in range(-6, 30, 2)]
    for border in (2.0 ** 30, 2.0 ** 31):
        rows += [sign * (border + 64.0 * torch.randint(-8, 9, (v,), generator=r)) for sign in (1, -1)]
    for mask in (-1e4, -1e9, -1e20, 1e9):
        row = torch.full((v,), mask)
        row[torch.randint(0, v, (5,), generator=r)] = torch.randn(5, generator=r)
        rows.append(row)
    x = torch.stack(rows).to(DT[dtype])
    t = torch.randint(0, v, (len(rows),), generator=r)
    t[::2] = x[::2].argmax(-1)
    for top in (0, 9):
        scoring_ref.check_logprobs(ops.token_logprobs(x.cuda(), t.cuda(), top), x, t, top)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_token_logprobs_sorted_rows(lib, dtype):
    """Rows that rise or fall along the vocabulary (every value a new maximum, or none), and large ones last."""
    from minitp_b200 import ops

    v = 50001
    up = torch.linspace(-30, 30, v)
    late = torch.full((v,), -5.0)
    late[-70:] = torch.linspace(3, 4, 70)
    x = torch.stack([up, up.flip(0), late, late.flip(0)]).to(DT[dtype])
    t = torch.tensor([v - 1, 0, v - 5, 3])
    for top in (0, 1, 20, 64):
        scoring_ref.check_logprobs(ops.token_logprobs(x.cuda(), t.cuda(), top), x, t, top)


def test_token_logprobs_shapes_and_strides(lib):
    """Leading axes, padded and expanded rows, an odd start of the data, targets of any stride."""
    from minitp_b200 import ops

    r = _gen(3)
    for dtype in DT.values():
        x = (torch.randn(2, 3, 1001, generator=r) * 2).to(dtype).cuda()
        t = torch.randint(0, 1001, (2, 3), generator=r).cuda()
        want = ops.token_logprobs(x.view(6, -1), t.view(-1), 4)
        got = ops.token_logprobs(x, t, 4)
        assert got[0].shape == got[1].shape == (2, 3) and got[2].shape == got[3].shape == (2, 3, 4)
        wide = torch.full((2, 3, 1100), 50.0, dtype=dtype, device="cuda")
        wide[..., 77:1078] = x
        tt = torch.empty(3, 2, dtype=torch.int64, device="cuda").T
        tt.copy_(t)
        for g in (got, ops.token_logprobs(wide[..., 77:1078], tt, 4), ops.token_logprobs(x.transpose(0, 1).contiguous().transpose(0, 1), t, 4),
                  ops.token_logprobs(x.transpose(1, 2).contiguous().transpose(1, 2), t, 4)):
            # (a row's sums are added in an order that goes by its place in memory)
            g = [a.reshape(b.shape) for a, b in zip(g, want)]
            scoring_ref.check_logprobs(g, x.view(6, -1), t.view(-1), 4)
        one = ops.token_logprobs(x[0, :1].expand(4, 1001), t.view(-1)[:4], 2)
        scoring_ref.check_logprobs(one, x[0, :1].expand(4, 1001), t.view(-1)[:4], 2)
        single = ops.token_logprobs(x[1, 2], t[1, 2], 3)
        assert single[0].shape == () and single[2].shape == (3,)
        scoring_ref.check_logprobs([a[None] for a in single], x[1, 2:], t[1, 2:], 3)
        none = ops.token_logprobs(x[:0], t[:0], 3)
        assert none[0].shape == (0, 3) and none[3].shape == (0, 3, 3)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("v,top", [(1000, 0), (9001, 5)])
def test_token_logprobs_offsets_past_32_bits(lib, dtype, v, top):
    """Rows that lie more than 2^31 elements apart."""
    from minitp_b200 import ops

    r = _gen(16)
    ld = 2 ** 30 + 8
    x = (torch.randn(4, v, generator=r) * 2).to(DT[dtype]).cuda()
    t = torch.randint(0, v, (4,), generator=r).cuda()
    wide = torch.empty(3 * ld + v, dtype=DT[dtype], device="cuda").as_strided((4, v), (ld, 1))
    wide.copy_(x)
    scoring_ref.check_logprobs(ops.token_logprobs(wide, t, top), x, t, top)


def test_token_logprobs_refusals(lib):
    from minitp_b200 import _lib, ops

    x, t = torch.zeros(2, 10, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    for args, match in [((x, t.int(), 2), "targets"), ((x, t[:1], 2), "targets"), ((x, t, 65), "alternatives"),
                        ((x, t, -1), "alternatives"), ((x.half(), t, 2), "unsupported dtype"), ((x, t.cpu(), 2), "CUDA"),
                        ((x[:, :0], t, 0), "vocabulary")]:
        with pytest.raises(_lib.MinitpB200Error, match=match):
            ops.token_logprobs(*args)


def test_token_logprobs_of_shards(lib):
    """Blocks of a vocabulary's shards (even, uneven, one empty) join to the whole call's result, in any order."""
    from minitp_b200 import ops

    r = _gen(21)
    for rows, v, top, cuts in [(5, 1000, 7, [0, 500, 1000]), (3, 10, 12, [0, 4, 7, 10, 10]), (70, 60000, 20, [0, 20000, 40000, 60000]),
                               (2, 3, 1, [0, 1, 2, 3, 3])]:
        for dtype in DT.values():
            x = (torch.randn(rows, v, generator=r) * 3).to(dtype)
            t = torch.randint(0, v, (rows,), generator=r)
            plan = max(b - a for a, b in zip(cuts, cuts[1:]))
            blocks = [ops.logprobs_block(x[:, a:b].cuda(), t.cuda(), top, a, plan) for a, b in zip(cuts, cuts[1:])]
            for order in (blocks, blocks[::-1]):
                got = ops.logprobs_join(torch.stack(order), t.cuda(), (rows,), top, plan, dtype)
                scoring_ref.check_logprobs(got, x, t, top)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_token_logprobs_joined_from_many_lists(lib, dtype):
    """Few long rows with many alternatives, and shards of every kind: more candidates than are ranked at once, among
    them runs of equal values and rows with fewer tokens than alternatives."""
    from minitp_b200 import ops

    r = _gen(77)
    v, top = 200003, 64
    x = (torch.randn(6, v, generator=r) * 3).to(DT[dtype])
    x[1] = torch.randint(-3, 3, (v,), generator=r).to(DT[dtype])
    x[2] = 0.0
    x[3] = -math.inf
    x[3, torch.randint(0, v, (40,), generator=r)] = 1.0
    x[4, 100000:] = -math.inf
    x[5, :4000] = 7.5
    t = torch.randint(0, v, (6,), generator=r)
    scoring_ref.check_logprobs(ops.token_logprobs(x.cuda(), t.cuda(), top), x, t, top)
    cuts = list(range(0, v, 6251)) + [v]
    blocks = [ops.logprobs_block(x[:, a:b].cuda(), t.cuda(), top, a, 6251) for a, b in zip(cuts, cuts[1:])]
    scoring_ref.check_logprobs(ops.logprobs_join(torch.stack(blocks), t.cuda(), (6,), top, 6251, DT[dtype]), x, t, top)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("v", [1, 9, 500, 4096, 8192])
def test_token_logprobs_many_short_rows(lib, dtype, v):
    """More rows than CTAs, of one tile each; every start in memory."""
    from minitp_b200 import ops

    r = _gen(v)
    wide = (torch.randn(3001, v + 3, generator=r) * 3).to(DT[dtype])
    wide[::5, ::3] = -math.inf
    for off in (0, 1, 3):
        x = wide[:, off:off + v]
        t = torch.randint(0, v, (3001,), generator=r)
        for top in (0, 3, 64):
            scoring_ref.check_logprobs(ops.token_logprobs(wide.cuda()[:, off:off + v], t.cuda(), top), x, t, top)


def test_token_logprobs_captured_and_on_another_stream(lib):
    from minitp_b200 import ops

    r = _gen(30)
    x = torch.randn(6, 30000, generator=r).cuda()
    t = torch.randint(0, 30000, (6,), generator=r).cuda()
    ops.token_logprobs(x, t, 8)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.token_logprobs(x, t, 8)
    side = torch.cuda.Stream()
    for _ in range(2):
        x.copy_(torch.randn(6, 30000, generator=r) * 4)
        t.copy_(torch.randint(0, 30000, (6,), generator=r))
        g.replay()
        scoring_ref.check_logprobs(out, x, t, 8)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = ops.token_logprobs(x, t, 8)
        side.synchronize()
        for a, b in zip(out, other):
            assert torch.equal(a, b)


def test_status_is_clean(lib):
    import ctypes

    s = ctypes.c_uint32(7)
    assert lib.mtpb_scoring_status(ctypes.byref(s)) == 0 and s.value == 0
