"""Workloads of packed prompt attention and token log-probabilities, with their plain forms.

Two operators of scoring prompts:

* ``prompt``    causal attention of whole prompts of different lengths, packed one
                behind the other, with grouped heads (``ops.prompt_attention``);
* ``logprobs``  log-probabilities of given tokens, the entropy of each row and its
                top alternatives (``ops.token_logprobs``).

``own`` chooses between the package's kernels and the plain form below, which is
elementary torch in 32 bits (the sums over a vocabulary in 64).
"""

import math

import torch

own = False

DT = {"fp32": torch.float32, "bf16": torch.bfloat16}

# (query heads, KV heads, head dim): the tiny, 0.5B and 7B shapes on one rank, and
# their shares on 2 to 8 ranks
HEADS = [(4, 2, 16), (14, 2, 64), (7, 1, 64), (28, 4, 128), (7, 1, 128), (4, 1, 128), (8, 4, 32)]


def _prompt(name, count, longest, hq, hkv, hd, dtype):
    return {"name": name, "op": "prompt", "count": count, "longest": longest, "hq": hq, "hkv": hkv, "hd": hd,
            "dtype": dtype}


def _logprobs(name, rows, vocab, top, masked, dtype):
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "top": top, "masked": masked,
            "dtype": dtype}


def listed():
    return [
        # three prompts of the tiny model: the latency of one call
        _prompt("prompt-tiny", 3, 23, 4, 2, 16, "fp32"),
        # one prompt of 128 tokens, 0.5B heads
        _prompt("prompt-128", 1, 128, 14, 2, 64, "bf16"),
        # one prompt of 1024 tokens, a rank's heads of the 7B shape on four
        _prompt("prompt-1024", 1, 1024, 7, 1, 128, "bf16"),
        # many short prompts of a scored data set, 0.5B heads
        _prompt("prompt-64-ragged", 64, 509, 14, 2, 64, "bf16"),
        # odd lengths in fp32
        _prompt("prompt-ragged-fp32", 5, 701, 8, 4, 32, "fp32"),
        # a batch of long documents, 7B heads
        _prompt("prompt-12-long", 12, 4096, 28, 4, 128, "bf16"),
        # one prompt as long as the 7B shape takes them
        _prompt("prompt-32768", 1, 32768, 28, 4, 128, "bf16"),
        # a decode step of the tiny model
        _logprobs("logprobs-tiny", 1, 1000, 4, False, "fp32"),
        # a decode step of four rows, 0.5B vocabulary
        _logprobs("logprobs-4-rows", 4, 151936, 5, False, "bf16"),
        # an odd vocabulary in fp32, every seventh token banned
        _logprobs("logprobs-300-fp32", 300, 151937, 8, True, "fp32"),
        # a piece of a scored batch with 20 alternatives a token, 7B vocabulary
        _logprobs("logprobs-512-top20", 512, 152064, 20, False, "bf16"),
        # the perplexity of a batch: no alternatives
        _logprobs("logprobs-4096", 4096, 151936, 0, False, "bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    case = _draw(rng)
    del case["name"]
    return case


def _draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if rng.choice(["prompt", "logprobs"]) == "logprobs":
        vocab = rng.choice([_log(rng, 50, 200000), 151936, 152064, 75968])
        # at most the bytes of the largest listed case
        most = 4096 * 151936 // (vocab * (1 if dtype == "bf16" else 2))
        rows = _log(rng, 1, max(1, min(8192, most)))
        top = rng.choice([0, 1, 5, _log(rng, 1, 64)])
        return _logprobs("", rows, vocab, min(top, vocab), rng.random() < 0.3, dtype)
    hq, hkv, hd = rng.choice(HEADS)
    count = _log(rng, 1, 64)
    longest = _log(rng, 1, 16384)
    # at most a thirtieth of the score entries of the largest listed case, and its tokens
    while count > 1 and hq * sum(n * n for n in _lengths(count, longest)) > 10 ** 9:
        count //= 2
    if hq * longest * longest > 10 ** 9:
        longest = int((10 ** 9 / hq) ** 0.5)
    return _prompt("", count, longest, hq, hkv, hd, dtype)


def _lengths(count, longest):
    """Ragged lengths that go by the case alone: the longest, then others down to a single token
    (and an empty prompt for every eleventh)."""
    return [0 if i % 11 == 10 else longest - (i * 3737) % longest for i in range(count)]


def _banned(case):
    """Vocabulary ids that a masked case bans: every seventh."""
    return slice(3, None, 7)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DT[case["dtype"]]
    s = {"case": case}
    if case["op"] == "logprobs":
        rows, v = case["rows"], case["vocab"]
        x = torch.empty(rows, v, dtype=dt, device="cuda")
        for i in range(0, rows, 512):
            x[i:i + 512] = torch.randn(min(512, rows - i), v, generator=g, device="cuda") * 2.5
        # half of the tokens are the likeliest of their row, half any that is not banned
        ids = torch.randint(0, v, (rows,), generator=g, device="cuda")
        if case["masked"]:
            x[:, _banned(case)] = -torch.inf
            ids = torch.where((ids % 7 == 3), ids - 1, ids)
        likely = torch.rand(rows, generator=g, device="cuda") < 0.5
        s["targets"] = torch.where(likely, x.argmax(-1), ids)
        s["logits"] = x
        return s
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    lengths = _lengths(case["count"], case["longest"])
    starts = [0]
    for n in lengths:
        starts.append(starts[-1] + n)
    # one projection's output, whose parts are q, k and v
    qkv = torch.randn(starts[-1], hq + 2 * hkv, hd, generator=g, device="cuda")
    qkv[:, :hq] *= 1.5
    s["qkv"] = qkv = qkv.to(dt)
    s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    s["seq_starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["lengths"] = lengths
    return s


# ------------------------------------------------------------------ plain forms
def _plain_prompt(q, k, v, lengths):
    hq, hd = q.shape[1:]
    hkv = k.shape[1]
    per = hq // hkv
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    start = 0
    for n in lengths:
        kf = k[start:start + n].float().permute(1, 2, 0)  # [hkv, hd, n]
        vf = v[start:start + n].float().transpose(0, 1)
        block = max(1, min(n, 2 ** 28 // max(1, hq * n)))  # tokens whose scores are held at once
        for i in range(0, n, block):
            e = min(n, i + block)
            qf = q[start + i:start + e].float().view(e - i, hkv, per, hd).permute(1, 2, 0, 3)
            sc = qf.reshape(hkv, per * (e - i), hd) @ kf[:, :, :e] / math.sqrt(hd)
            sc = sc.view(hkv, per, e - i, e)
            seen = torch.arange(e, device=q.device) <= torch.arange(i, e, device=q.device)[:, None]
            sc = torch.where(seen, sc, -torch.inf)
            sc = (sc - sc.amax(-1, keepdim=True)).exp()
            total = sc.sum(-1, keepdim=True)
            o = (sc.view(hkv, per * (e - i), e) @ vf[:, :e]).view(hkv, per, e - i, hd) / total
            out[start + i:start + e] = o.permute(2, 0, 1, 3).reshape(e - i, hq, hd).to(q.dtype)
        start += n
    return out


def _plain_logprobs(logits, targets, top):
    parts = []
    for i in range(0, logits.shape[0], 512):
        x = logits[i:i + 512]
        m = x.amax(-1, keepdim=True).double()
        d = x.double() - m
        e = d.exp()
        total = e.sum(-1)
        logz = total.log()
        entropy = logz - torch.where(e > 0, e * d, 0.0).sum(-1) / total
        logprob = d.gather(1, targets[i:i + 512, None]).squeeze(1) - logz
        best = at = None
        if top:
            best, at = x.float().sort(dim=-1, descending=True, stable=True)
            best, at = best[:, :top], at[:, :top]
            best = best.double() - m - logz[:, None]
            at = torch.where(torch.isneginf(best), 0, at)
            best = best.float()
        parts.append((logprob.float(), entropy.float(), best, at))
    return tuple(None if p[0] is None else torch.cat(p) for p in zip(*parts))


def run(s):
    case = s["case"]
    if own:
        from minitp_b200 import ops
    if case["op"] == "prompt":
        if own:
            return ops.prompt_attention(s["q"], s["k"], s["v"], s["seq_starts"])
        return _plain_prompt(s["q"], s["k"], s["v"], s["lengths"])
    fn = ops.token_logprobs if own else _plain_logprobs
    logprobs, entropy, top_logprobs, top_ids = fn(s["logits"], s["targets"], case["top"])
    out = {"logprobs": logprobs, "entropy": entropy}
    if case["top"]:
        out["top_logprobs"], out["top_ids"] = top_logprobs, top_ids
    return out


def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "logprobs":
        rows = case["rows"]
        # logits and targets in; two values and the alternatives out; a maximum, an exponential, a product and two
        # sums a value
        return {"bytes": float(rows * (case["vocab"] * es + 8 + 8 + 12 * case["top"])),
                "flops": 5.0 * rows * case["vocab"]}
    lengths = _lengths(case["count"], case["longest"])
    heads, hd = 2 * case["hq"] + 2 * case["hkv"], case["hd"]
    return {"bytes": float(sum(lengths) * heads * hd * es + 4 * (case["count"] + 1)),
            "flops": 4.0 * case["hq"] * hd * sum(n * (n + 1) // 2 for n in lengths)}


# ------------------------------------------------------------------ from the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        logprobs, entropy, tops = [], [], []
        for i in range(0, case["rows"], 256):
            logp = torch.log_softmax(s["logits"][i:i + 256].double(), -1)
            logprobs.append(logp.gather(1, s["targets"][i:i + 256, None]).squeeze(1))
            entropy.append(torch.special.entr(logp.exp()).sum(-1))
            if case["top"]:
                tops.append(logp.topk(case["top"], dim=-1).values)
        out = {"logprobs": torch.cat(logprobs), "entropy": torch.cat(entropy)}
        if case["top"]:
            out["top_logprobs"], out["top_ids"] = torch.cat(tops), None
        return out
    per = case["hq"] // case["hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for a, b in zip(s["seq_starts"].tolist(), s["seq_starts"].tolist()[1:]):
        for h in range(case["hq"]):
            keys, vals = s["k"][a:b, h // per].double(), s["v"][a:b, h // per].double()
            for i in range(a, b, 4096):
                e = min(b, i + 4096)
                sc = (s["q"][i:e, h].double() @ keys[:e - a].T) * case["hd"] ** -0.5
                hidden = torch.ones_like(sc, dtype=torch.bool).triu(i - a + 1)
                out[i:e, h] = torch.softmax(sc.masked_fill(hidden, -torch.inf), -1) @ vals[:e - a]
    return out
