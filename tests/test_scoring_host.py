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
                          (dict(vh=-64), "strides"), (dict(n=1, total=1 << 27), "rows")]:
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
