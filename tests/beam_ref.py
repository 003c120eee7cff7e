"""Plain 64-bit implementations of beam selection, cache reordering and shared-prefix attention."""

import math

import torch

EPS32 = 2.0 ** -24  # half a step of fp32, relative
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def totals(logits, scores, finished=None, eos=None):
    """[G, W, V] fp64 candidate scores on the CPU; -inf where there is no candidate."""
    x = logits.detach().cpu().double()
    s = scores.detach().cpu().double()
    g, w, v = x.shape
    out = torch.full((g, w, v), -math.inf, dtype=torch.float64)
    for i in range(g):
        for b in range(w):
            if finished is not None and bool(finished[i, b]):
                out[i, b, eos] = s[i, b]
                continue
            row = x[i, b].clone()
            row[torch.isnan(row)] = -math.inf
            if math.isnan(s[i, b]) or s[i, b] == -math.inf or row.max() == -math.inf:
                continue
            if row.max() == math.inf:
                hot = row == math.inf
                out[i, b, hot] = s[i, b] - math.log(int(hot.sum()))
            else:
                row -= row.max()  # first: next to the type's lowest value the logarithm would be lost
                out[i, b] = s[i, b] + row - torch.logsumexp(row, 0)
    if finished is not None:
        out[torch.isnan(out)] = -math.inf
    return out


def select(logits, scores, k, finished=None, eos=None):
    """(scores fp64, parents, tokens, finished) of the k best, by the definition."""
    t = totals(logits, scores, finished, eos)
    g, w, v = t.shape
    best = torch.full((g, k), -math.inf, dtype=torch.float64)
    par = torch.zeros(g, k, dtype=torch.int64)
    tok = torch.full((g, k), 0 if eos is None else eos, dtype=torch.int64)
    order = torch.sort(t.view(g, -1), dim=-1, descending=True, stable=True)
    for i in range(g):
        for j in range(min(k, w * v)):
            if order.values[i, j] == -math.inf:
                break
            best[i, j] = order.values[i, j]
            par[i, j], tok[i, j] = divmod(int(order.indices[i, j]), v)
    done = None
    if eos is not None:
        old = finished.cpu() if finished is not None else torch.zeros(g, w, dtype=torch.bool)
        done = (tok == eos) | old.gather(1, par)
    return best, par, tok, done


def select_tolerance(v, best):
    """fp32 sum of the exponentials, each off by a few half steps, added at most V/256 + 40 deep;
    then the total's rounding to fp32."""
    finite = best[torch.isfinite(best)]
    big = float(finite.abs().max()) if finite.numel() else 0.0
    return (v / 256 + 40) * EPS32 + 2 * EPS32 * big


def check_select(got, logits, scores, k, finished=None, eos=None):
    """`got` is a selection by the definition: sorted, of distinct candidates, each with its own total, and
    none better left out; where neighbours are further apart than the tolerance the ids are the definition's."""
    out, par, tok, done = (None if x is None else x.cpu() for x in got)
    best, wpar, wtok, wdone = select(logits, scores, k, finished, eos)
    v = logits.shape[-1]
    tol = select_tolerance(v, best)
    assert out.dtype == torch.float32 and par.dtype == tok.dtype == torch.int64
    assert torch.equal(torch.isinf(out), torch.isinf(best))
    fine = torch.isfinite(best)
    assert float((out.double() - best)[fine].abs().max() if fine.any() else 0.0) <= tol
    t = totals(logits, scores, finished, eos)
    for g in range(best.shape[0]):
        seen = set()
        for j in range(k):
            if not fine[g, j]:
                assert (int(par[g, j]), int(tok[g, j])) == (int(wpar[g, j]), int(wtok[g, j]))
                continue
            at = (int(par[g, j]), int(tok[g, j]))
            assert at not in seen
            seen.add(at)
            if at != (int(wpar[g, j]), int(wtok[g, j])):
                # only a candidate of another beam within the rounding may stand here
                assert abs(float(t[g, at[0], at[1]]) - float(best[g, j])) <= 2 * tol
                assert at[0] != int(wpar[g, j])
    if eos is None:
        assert done is None
    else:
        old = finished.cpu() if finished is not None else torch.zeros(scores.shape, dtype=torch.bool)
        assert torch.equal(done, (tok == eos) | old.gather(1, par))


def check_totals(got, logits, scores, k):
    """Every place holds the total of the candidate that it names, and is the place's best, each within
    `select_tolerance` of its own size (one candidate of -1e9 loosens nothing for the others)."""
    out, par, tok = (x.cpu() for x in got[:3])
    best, wpar, wtok, _ = select(logits, scores, k)
    t = totals(logits, scores)
    v = logits.shape[-1]
    for g in range(best.shape[0]):
        assert len({(int(p), int(x)) for p, x, b in zip(par[g], tok[g], best[g]) if b > -math.inf}) == \
            int((best[g] > -math.inf).sum())
        for j in range(k):
            at, want = (int(par[g, j]), int(tok[g, j])), float(best[g, j])
            if want == -math.inf:
                assert float(out[g, j]) == want and at == (int(wpar[g, j]), int(wtok[g, j]))
                continue
            tol = select_tolerance(v, best[g, j])
            assert abs(float(out[g, j]) - want) <= tol, (g, j, float(out[g, j]), want)
            assert abs(float(t[g, at[0], at[1]]) - want) <= 2 * tol


def reorder(cache, parents, lengths):
    """The reordered copy of one [G*W, hkv, cap, hd] cache."""
    out = cache.clone()
    g, w = parents.shape
    for i in range(g):
        for b in range(w):
            p = int(parents[i, b])
            if 0 <= p < w:
                n = int(lengths[i * w + p])
                out[i * w + b, :, :n] = cache[i * w + p, :, :n]
    return out


def attend(q, kp, vp, plen, kc, vc, clen, hq, hkv):
    """(out fp64 [N, T, hq*hd], tolerance of the same shape) on the CPU.

    Tolerance, per value, for a kernel that adds products in fp32 and (bf16) rounds probabilities:
    a score is off by (hd + 4) half steps of sum |q_i k_i| / sqrt(hd); a probability by twice that
    and (keys + 64) half steps of the sums; the output by that times max |v|, plus (bf16) a half step
    of bf16 of sum p |v| for the probabilities and of the value itself for the result."""
    q, kp, vp, kc, vc = (x.detach().cpu() for x in (q, kp, vp, kc, vc))
    n, t, _ = q.shape
    g, hd, per = kp.shape[0], kp.shape[-1], hq // hkv
    w = n // g
    half = HALF[q.dtype]
    out = torch.zeros(n, t, hq, hd, dtype=torch.float64)
    tol = torch.zeros(n, t, hq, hd, dtype=torch.float64)
    for r in range(n):
        pl = max(0, min(int(plen[r // w]), kp.shape[2]))
        cl = max(0, min(int(clen[r]), kc.shape[2]))
        for h in range(hq):
            keys = torch.cat([kp[r // w, h // per, :pl], kc[r, h // per, :cl]]).double()
            vals = torch.cat([vp[r // w, h // per, :pl], vc[r, h // per, :cl]]).double()
            for i in range(t):
                seen = pl + max(0, cl - (t - 1 - i))
                if seen == 0:
                    continue
                qs = q[r, i].view(hq, hd)[h].double()
                s = keys[:seen] @ qs / math.sqrt(hd)
                p = torch.softmax(s, 0)
                o = p @ vals[:seen]
                out[r, i, h] = o
                off = (hd + 4) * EPS32 * float((keys[:seen].abs() @ qs.abs()).max()) / math.sqrt(hd)
                rel = 2 * off + (seen + 64) * EPS32
                tol[r, i, h] = rel * float(vals[:seen].abs().max()) + half * o.abs() * 1.01
                if q.dtype == torch.bfloat16:
                    tol[r, i, h] += half * (p @ vals[:seen].abs()) * 1.01
    return out.view(n, t, -1), tol.view(n, t, -1)
