"""Plain 64-bit implementations of packed prompt attention and token log-probabilities."""

import math

import torch

from tests.beam_ref import EPS32, HALF


def attend(q, k, v, starts, first=0):
    """(out fp64 [n, hq, hd], tolerance of the same shape) on the CPU; `starts` a list.

    Tolerance, per value, for a kernel that adds products in fp32 and (bf16) rounds probabilities: a score is off
    by (hd + 4) half steps of sum |q_i k_i| / sqrt(hd); a probability by twice that and (keys + 64) half steps of
    the sums; the output by that times max |v| (2^-14 of it more in bf16, whose exponentials may come from a
    cubic), plus (bf16) a half step of bf16 of sum p |v| for the probabilities and of the value itself for the
    result, 1.01 for products of the two."""
    q, k, v = (x.detach().cpu().double() if x.dtype == torch.float32 else x.detach().cpu() for x in (q, k, v))
    low = q.dtype == torch.bfloat16
    half = HALF[torch.bfloat16] if low else HALF[torch.float32]
    q, k, v = q.double(), k.double(), v.double()
    n, hq, hd = q.shape
    per = hq // k.shape[1]
    out = torch.zeros(n, hq, hd, dtype=torch.float64)
    tol = torch.zeros(n, hq, hd, dtype=torch.float64)
    for a, b in zip(starts, starts[1:]):
        lo, hi = max(a, first), min(b, first + n)
        if lo >= hi:
            continue
        hidden = torch.arange(a, hi)[None] > torch.arange(lo, hi)[:, None]
        for h in range(hq):
            qs, keys, vals = q[lo - first:hi - first, h], k[a:hi, h // per], v[a:hi, h // per]
            s = (qs @ keys.T / math.sqrt(hd)).masked_fill(hidden, -math.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.where(hidden, 0.0, (s - torch.where(torch.isneginf(top), 0.0, top)).exp())
            total = p.sum(-1, keepdim=True)
            p = torch.where(total == 0, 0.0, p / total)
            # a product with an unseen value is left out, whatever the value
            finite = torch.nan_to_num(vals, 0.0, 0.0, 0.0)
            o = p @ finite
            for j in torch.nonzero(~torch.isfinite(vals).all(-1)).flatten().tolist():
                wrong = torch.where(torch.isfinite(vals[j]), 0.0, vals[j])
                o = torch.where((~hidden[:, j] & (total[:, 0] != 0))[:, None], o + p[:, j, None] * wrong, o)
            out[lo - first:hi - first, h] = o
            mag = torch.where(hidden, 0.0, torch.nan_to_num(qs.abs() @ keys.abs().T, 0.0, 0.0, 0.0)).amax(-1)
            rel = 2 * (hd + 4) * EPS32 * mag / math.sqrt(hd) + (hi - a + 64) * EPS32 + (2.0 ** -14 if low else 0.0)
            seen_max = torch.where(hidden, 0.0, finite.abs().amax(-1)).amax(-1)
            t = (rel * seen_max)[:, None] + half * o.abs() * 1.01
            if low:
                t = t + half * (p @ finite.abs()) * 1.01
            tol[lo - first:hi - first, h] = t
    return out, tol


def logprobs(logits, targets, top):
    """(logprobs, entropy, top_logprobs, top_ids) in fp64 on the CPU, by the definition, rows [n, V]."""
    x = logits.detach().cpu().double()
    n, v = x.shape
    x = torch.where(torch.isnan(x), -math.inf, x)
    m = x.amax(-1, keepdim=True)
    d = torch.where(x == m, 0.0, x - torch.where(torch.isinf(m) & (x != m) & (m < 0), 0.0, m))
    d = torch.where(torch.isneginf(x), -math.inf, d)
    e = d.exp()
    total = e.sum(-1, keepdim=True)
    none = total == 0
    logz = torch.where(none, 0.0, total.log())
    logp = torch.where(none, -math.inf, d - logz)
    p = logp.exp()
    entropy = torch.where(p > 0, -p * logp, 0.0).sum(-1)
    lp = None
    if targets is not None:
        t = targets.detach().cpu()
        ok = (t >= 0) & (t < v)
        lp = torch.where(ok, logp.gather(1, t.clamp(0, v - 1)[:, None])[:, 0], math.nan)
    best = torch.full((n, top), -math.inf, dtype=torch.float64)
    ids = torch.zeros(n, top, dtype=torch.int64)
    if top:
        keep = min(top, v)
        order = torch.where(torch.isnan(logits.detach().cpu().double()), -math.inf, logits.detach().cpu().double())
        at = (order + 0.0).sort(dim=-1, descending=True, stable=True).indices[:, :keep]
        best[:, :keep] = logp.gather(1, at)
        live = ~torch.isneginf(order.gather(1, at))
        ids[:, :keep] = torch.where(live, at, 0)
        best[:, :keep] = torch.where(live, best[:, :keep], -math.inf)
    return lp, entropy, best, ids


def check_logprobs(got, logits, targets, top):
    """`got` against the definition. A sum of exponentials, each off by a few half steps, is added at most
    V / 256 + 40 deep; a log-probability is off by that and its own rounding, and the entropy, whose terms
    carry the logarithm as a factor, by that times (2 + H)."""
    lp, ent, best, ids = logprobs(logits, targets, top)
    v = logits.shape[-1]
    base = (v / 256 + 40) * EPS32

    def near(a, want, tol):
        a = a.detach().cpu()
        assert a.dtype == torch.float32 and a.shape == want.shape
        a = a.double()
        assert torch.equal(torch.isnan(a), torch.isnan(want))
        want = torch.where(torch.isinf(want.float()), want.float().double(), want)  # (2 x fp32's range: -inf there)
        assert torch.equal(torch.isinf(a), torch.isinf(want))
        fine = torch.isfinite(want)
        off = (a - want).abs()[fine] - tol[fine]
        assert off.numel() == 0 or float(off.max()) <= 0, float(off.max())

    if targets is None:
        assert got[0] is None
    else:
        near(got[0], lp, base + 2 * EPS32 * lp.abs())
    near(got[1], ent, base * (2 + ent))
    if top:
        assert got[3].dtype == torch.int64
        assert torch.equal(got[3].detach().cpu(), ids)
        near(got[2], best, base + 2 * EPS32 * best.abs())
    else:
        assert got[2] is None and got[3] is None
