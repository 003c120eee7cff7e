"""Workloads of the beam-search and shared-prefix operators, with their plain forms.

Three operators of batched decoding:

* ``select``   one step of beam search: log-softmax over the vocabulary, running
               scores, the best k of (beams x vocabulary) per prompt
               (``ops.beam_select``);
* ``reorder``  the KV cache rows of every layer follow the chosen beams, in place
               (``ops.reorder_cache_``);
* ``attend``   attention of rows that share a prefix: row n of group g sees the
               group's prefix cache and its own cache (``ops.shared_prefix_attention``).

``own`` chooses between the package's kernels and the plain form below, which is
elementary torch in 32 bits (the selection in 64: candidates of different beams
are compared by their sums).
"""

import math

import torch

own = False

DT = {"fp32": torch.float32, "bf16": torch.bfloat16}

# (query heads, KV heads, head dim): the tiny, 0.5B and 7B shapes on one rank, and
# their shares on 2 to 8 ranks
HEADS = [(4, 2, 16), (14, 2, 64), (7, 1, 64), (28, 4, 128), (7, 1, 128), (4, 1, 128), (8, 4, 32)]


def _select(name, groups, beams, vocab, k, dtype, eos):
    return {"name": name, "op": "select", "groups": groups, "beams": beams, "vocab": vocab, "k": k, "dtype": dtype,
            "eos": eos}


def _reorder(name, layers, groups, beams, hkv, hd, cap, length, dtype):
    return {"name": name, "op": "reorder", "layers": layers, "groups": groups, "beams": beams, "hkv": hkv, "hd": hd,
            "cap": cap, "length": length, "dtype": dtype}


def _attend(name, groups, width, tokens, hq, hkv, hd, pcap, prefix, cap, length, dtype):
    return {"name": name, "op": "attend", "groups": groups, "width": width, "tokens": tokens, "hq": hq, "hkv": hkv,
            "hd": hd, "pcap": pcap, "prefix": prefix, "cap": cap, "length": length, "dtype": dtype}


def listed():
    return [
        # one prompt of the tiny model, 4 beams: the latency of one call
        _select("select-tiny", 1, 4, 1000, 4, "fp32", False),
        # one prompt of the 0.5B shape, 4 beams, no end token
        _select("select-4-beams", 1, 4, 151936, 4, "bf16", False),
        # eight prompts of the 7B shape, 8 beams each, some finished
        _select("select-8x8-eos", 8, 8, 152064, 8, "bf16", True),
        # a large batch in fp32, an odd vocabulary, twice as many candidates as beams
        _select("select-32x16-fp32", 32, 16, 151937, 32, "fp32", True),
        # the tiny model's cache: a copy of a few kilobytes
        _reorder("reorder-tiny", 2, 1, 4, 2, 16, 32, 9, "fp32"),
        # the 0.5B shape half way through 128 new tokens, 4 beams
        _reorder("reorder-4-beams", 24, 1, 4, 2, 64, 128, 65, "bf16"),
        # the 7B shape, eight prompts of 8 beams, 256 new tokens nearly done
        _reorder("reorder-8x8", 28, 8, 8, 4, 128, 256, 250, "bf16"),
        # beam search on one prompt of 128 tokens, 0.5B heads: latency
        _attend("attend-4-beams", 1, 4, 1, 14, 2, 64, 128, 128, 128, 16, "bf16"),
        # ragged prefixes and own lengths down to nothing, fp32, odd sizes
        _attend("attend-ragged-fp32", 3, 5, 1, 4, 2, 16, 333, 333, 77, 77, "fp32"),
        # eight prompts of up to 1024 tokens, 8 beams each, 7B heads
        _attend("attend-8x8", 8, 8, 1, 28, 4, 128, 1024, 1024, 256, 250, "bf16"),
        # 64 requests behind one long system prompt, 7B heads
        _attend("attend-64-long", 1, 64, 1, 28, 4, 128, 16384, 16384, 512, 500, "bf16"),
        # the requests' own prompts after the shared one: many tokens a row
        _attend("attend-16x128-tokens", 1, 16, 128, 14, 2, 64, 4096, 4001, 160, 150, "bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    case = _draw(rng)
    del case["name"]
    return case


def _draw(rng):
    op = rng.choice(["select", "reorder", "attend"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "select":
        # at most the values of the largest listed case
        beams = _log(rng, 1, 32)
        vocab = rng.choice([_log(rng, 50, 200000), 151936, 152064, 75968])
        groups = _log(rng, 1, max(1, min(64, 512 * 151937 // (beams * vocab))))
        k = min(64, rng.choice([beams, beams, 2 * beams]))
        return _select("", groups, beams, vocab, k, dtype, rng.random() < 0.5)
    hq, hkv, hd = rng.choice(HEADS)
    if op == "reorder":
        layers, beams = _log(rng, 1, 32), _log(rng, 2, 32)
        cap = _log(rng, 4, 1024)
        row = layers * beams * hkv * cap * hd * (2 if dtype == "bf16" else 4)
        groups = _log(rng, 1, max(1, min(16, 1_800_000_000 // row)))
        return _reorder("", layers, groups, beams, hkv, hd, cap, rng.randint(1, cap), dtype)
    tokens = rng.choice([1, 1, 1, _log(rng, 2, 128)])
    width = _log(rng, 1, 64 if tokens == 1 else 16)
    pcap = _log(rng, 1, 16384 if tokens == 1 else 4096)
    cap = tokens + _log(rng, 1, 512)
    # at most the score entries of the largest listed case
    groups = _log(rng, 1, max(1, min(8, 120_000_000 // (width * tokens * hq * (pcap + cap)))))
    if width * tokens * hq * (pcap + cap) > 120_000_000:
        pcap = max(1, 120_000_000 // (width * tokens * hq) - cap)
    return _attend("", groups, width, tokens, hq, hkv, hd, pcap, rng.randint(1, pcap), cap, rng.randint(1, cap),
                   dtype)


def _lengths(count, longest):
    """Ragged lengths that go by the case alone: the longest, then shorter ones down to about half of it
    (and to none, for every seventh)."""
    return [0 if i % 7 == 6 else longest - (i * 37) % max(1, longest // 2) for i in range(count)]


def _parent_odds(beams):
    """How often each old beam (best first) is a new beam's parent."""
    edge = [(i / beams) ** (2 / 3) for i in range(beams + 1)]
    return [b - a for a, b in zip(edge, edge[1:])]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DT[case["dtype"]]
    s = {"case": case}

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    if case["op"] == "select":
        n, w, v = case["groups"], case["beams"], case["vocab"]
        s["logits"] = (randn(n, w, v) * 2.5).to(dt)
        s["scores"] = randn(n, w) * 2.0 - 20.0
        s["eos"] = v // 2 if case["eos"] else None
        s["finished"] = None
        if case["eos"]:
            s["finished"] = torch.rand(n, w, generator=g, device="cuda") < 0.25
        return s
    if case["op"] == "reorder":
        n, w = case["groups"], case["beams"]
        shape = (case["layers"], n * w, case["hkv"], case["cap"], case["hd"])
        s["k"] = torch.empty(shape, dtype=dt, device="cuda").normal_(generator=g)
        s["v"] = torch.empty(shape, dtype=dt, device="cuda").normal_(generator=g)
        s["k_layers"], s["v_layers"] = list(s["k"].unbind(0)), list(s["v"].unbind(0))
        u = torch.rand(n, w, generator=g, device="cuda")
        s["parents"] = (w * u ** 1.5).long().clamp_(max=w - 1)
        s["lengths"] = torch.tensor(_lengths(n, case["length"]), dtype=torch.int32,
                                    device="cuda").repeat_interleave(w)
        return s
    n, w, t = case["groups"], case["width"], case["tokens"]
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    s["q"] = (randn(n * w, t, hq * hd) * 1.5).to(dt)
    s["kp"], s["vp"] = (randn(n, hkv, case["pcap"], hd).to(dt) for _ in range(2))
    s["kc"], s["vc"] = (randn(n * w, hkv, case["cap"], hd).to(dt) for _ in range(2))
    s["prefix_lens"] = torch.tensor(_lengths(n, case["prefix"]), dtype=torch.int32, device="cuda")
    s["cache_lens"] = torch.tensor(_lengths(n * w, case["length"]), dtype=torch.int32, device="cuda")
    return s


# ------------------------------------------------------------------ plain forms
def _plain_select(logits, scores, k, finished, eos):
    n, w, v = logits.shape
    x = logits.double()
    x = torch.where(torch.isnan(x), -torch.inf, x)
    top = x.amax(-1, keepdim=True)
    x = torch.where(x == top, 0.0, x - top)
    logp = x - x.exp().sum(-1, keepdim=True).log()
    logp = torch.where(torch.isneginf(top), -torch.inf, logp)
    total = scores.double()[..., None] + logp
    if finished is not None:
        only = torch.arange(v, device=x.device) == eos
        kept = torch.where(only, scores.double()[..., None], -torch.inf)
        total = torch.where(finished[..., None], kept, total)
    flat = total.reshape(n, w * v)
    best, at = flat.sort(dim=-1, descending=True, stable=True)
    best, at = best[:, :k], at[:, :k]
    if w * v < k:
        best = torch.cat([best, best.new_full((n, k - w * v), -torch.inf)], -1)
        at = torch.cat([at, at.new_zeros((n, k - w * v))], -1)
    none = torch.isneginf(best)
    parents = torch.where(none, 0, at // v)
    tokens = torch.where(none, 0 if eos is None else eos, at % v)
    done = None if eos is None else (tokens == eos) | finished.gather(1, parents)
    return best.float(), parents, tokens, done


def _plain_reorder(k, v, parents, lengths):
    n, w = parents.shape
    rows = (torch.arange(n, device=parents.device)[:, None] * w + parents).reshape(-1)
    moves = torch.arange(k.shape[3], device=k.device) < lengths[rows][:, None]
    moves = moves[None, :, None, :, None]
    k.copy_(torch.where(moves, k[:, rows], k))
    v.copy_(torch.where(moves, v[:, rows], v))
    return k, v


def _plain_attend(q, kp, vp, prefix_lens, kc, vc, cache_lens, hq, hkv):
    n, t, _ = q.shape
    g, hd, pcap, cap = prefix_lens.numel(), kp.shape[-1], kp.shape[2], kc.shape[2]
    w, per = n // g, hq // hkv
    qf = q.float().view(n, t, hkv, per, hd).permute(0, 2, 1, 3, 4)  # [n, hkv, t, per, hd]
    seen_p = torch.arange(pcap, device=q.device) < prefix_lens[:, None]  # [g, pcap]
    ends = cache_lens[:, None] - (t - 1) + torch.arange(t, device=q.device)  # [n, t]
    seen_c = torch.arange(cap, device=q.device) < ends[:, :, None]  # [n, t, cap]
    qg = qf.reshape(g, w, hkv, t * per, hd).transpose(1, 2).reshape(g, hkv, w * t * per, hd)
    sp = qg @ kp.float().transpose(-1, -2) / math.sqrt(hd)
    sp = torch.where(seen_p[:, None, None], sp, -torch.inf)
    sp = sp.view(g, hkv, w, t * per, pcap).transpose(1, 2).reshape(n, hkv, t * per, pcap)
    sc = qf.reshape(n, hkv, t * per, hd) @ kc.float().transpose(-1, -2) / math.sqrt(hd)
    sc = torch.where(seen_c[:, None, :, None], sc.view(n, hkv, t, per, cap), -torch.inf).view(n, hkv, t * per, cap)
    top = torch.maximum(sp.amax(-1, keepdim=True), sc.amax(-1, keepdim=True))
    top = torch.where(torch.isneginf(top), 0.0, top)
    sp, sc = (sp - top).exp(), (sc - top).exp()
    total = sp.sum(-1, keepdim=True) + sc.sum(-1, keepdim=True)
    vpf = torch.where(seen_p[:, None, :, None], vp.float(), 0.0)
    vcf = torch.where(seen_c[:, -1][:, None, :, None], vc.float(), 0.0)
    op = sp.view(g, w, hkv, t * per, pcap).transpose(1, 2).reshape(g, hkv, w * t * per, pcap) @ vpf
    op = op.view(g, hkv, w, t * per, hd).transpose(1, 2).reshape(n, hkv, t * per, hd)
    o = (op + sc @ vcf) / torch.where(total > 0, total, 1.0)
    return o.view(n, hkv, t, per, hd).permute(0, 2, 1, 3, 4).reshape(n, t, hq * hd).to(q.dtype)


def run(s):
    case = s["case"]
    if own:
        from minitp_b200 import ops
    if case["op"] == "select":
        fn = ops.beam_select if own else _plain_select
        scores, parents, tokens, done = fn(s["logits"], s["scores"], case["k"], s["finished"], s["eos"])
        return {"scores": scores, "parents": parents, "tokens": tokens, "finished": done}
    if case["op"] == "reorder":
        if own:
            ops.reorder_cache_(s["k_layers"], s["v_layers"], s["parents"], s["lengths"])
        else:
            _plain_reorder(s["k"], s["v"], s["parents"], s["lengths"])
        return {"k": s["k"], "v": s["v"]}
    fn = ops.shared_prefix_attention if own else _plain_attend
    return fn(s["q"], s["kp"], s["vp"], s["prefix_lens"], s["kc"], s["vc"], s["cache_lens"], case["hq"], case["hkv"])


def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "select":
        rows = case["groups"] * case["beams"]
        # logits and scores in; scores, parents, tokens (and flags) out; a maximum, an exponential and two sums a value
        live = 0.75 if case["eos"] else 1.0
        return {"bytes": live * rows * case["vocab"] * es + 4 * rows + 20 * case["groups"] * case["k"],
                "flops": 4.0 * live * rows * case["vocab"]}
    if case["op"] == "reorder":
        w, odds = case["beams"], _parent_odds(case["beams"])
        moved = sum(1 - p for p in odds)
        read = sum(1 - (1 - p) ** (w - 1) for p in odds)
        tokens = sum(_lengths(case["groups"], case["length"]))
        return {"bytes": 2.0 * case["layers"] * tokens * case["hkv"] * case["hd"] * es * (moved + read), "flops": 0.0}
    n, t = case["groups"] * case["width"], case["tokens"]
    prefix, mine = _lengths(case["groups"], case["prefix"]), _lengths(n, case["length"])
    kv = 2.0 * case["hkv"] * case["hd"] * es * (sum(prefix) + sum(mine))
    pairs = sum(p * case["width"] * t for p in prefix) + sum(max(0, m - i) for m in mine for i in range(t))
    return {"bytes": kv + 2.0 * n * t * case["hq"] * case["hd"] * es, "flops": 4.0 * case["hq"] * case["hd"] * pairs}


# ------------------------------------------------------------------ from the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "reorder":  # copies: row by row, each value as it was
        parents, lengths, w = s["parents"].tolist(), s["lengths"].tolist(), case["beams"]
        was = {"k": s["k"], "v": s["v"]}
        now = {name: t.double() for name, t in was.items()}
        for g, chosen in enumerate(parents):
            for b, p in enumerate(chosen):
                src, n = g * w + p, lengths[g * w + p]
                for name in was:
                    now[name][:, g * w + b, :, :n] = was[name][:, src, :, :n].double()
        return now
    if case["op"] == "select":
        scores = []
        for logits, start, g in zip(s["logits"], s["scores"], range(case["groups"])):
            mine = []
            for b in range(case["beams"]):
                if s["finished"] is not None and bool(s["finished"][g, b]):
                    mine.append(start[b].double()[None])
                else:
                    mine.append(start[b].double() + torch.log_softmax(logits[b].double(), -1))
            mine = torch.cat(mine)
            if mine.numel() < case["k"]:
                mine = torch.cat([mine, mine.new_full((case["k"] - mine.numel(),), -torch.inf)])
            scores.append(mine.topk(case["k"]).values)
        return {"scores": torch.stack(scores), "parents": None, "tokens": None, "finished": None}
    hq, hkv, hd, t = case["hq"], case["hkv"], case["hd"], case["tokens"]
    n, per = case["groups"] * case["width"], hq // hkv
    out = torch.zeros(n, t, hq, hd, dtype=torch.float64, device="cuda")
    plen, clen = s["prefix_lens"].tolist(), s["cache_lens"].tolist()
    for r in range(n):
        g = r // case["width"]
        for h in range(hkv):
            keys = torch.cat([s["kp"][g, h, : plen[g]], s["kc"][r, h, : clen[r]]]).double()
            vals = torch.cat([s["vp"][g, h, : plen[g]], s["vc"][r, h, : clen[r]]]).double()
            qs = s["q"][r].view(t, hq, hd)[:, h * per : (h + 1) * per].double()
            sc = torch.einsum("tpd,kd->tpk", qs, keys) * hd ** -0.5
            last = plen[g] + clen[r] - t + torch.arange(t, device="cuda")  # the last key that token sees
            hidden = torch.arange(keys.shape[0], device="cuda") > last.clamp(min=plen[g] - 1)[:, None]
            pr = torch.softmax(sc.masked_fill(hidden[:, None], -torch.inf), -1)
            out[r, :, h * per : (h + 1) * per] = torch.nan_to_num(pr) @ vals
    return out.view(n, t, hq * hd)
