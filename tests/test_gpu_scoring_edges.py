"""Packed prompt attention and token log-probabilities where their schedules and masks have an edge."""

import ctypes
import math

import pytest
import torch

from tests import scoring_ref
from tests.test_gpu_scoring import DT, _close, _cuda_starts, _gen, _parts, _starts

pytestmark = pytest.mark.gpu


def _status_is_clean(lib):
    s = ctypes.c_uint32(7)
    assert lib.mtpb_scoring_status(ctypes.byref(s)) == 0 and s.value == 0


# ------------------------------------------------------------------ log-probabilities
def _check_some(got, x, t, top, step=13):
    """Every `step`-th row, and the last, against the definition."""
    at = torch.tensor(sorted({*range(0, x.shape[0], step), x.shape[0] - 1}), device=x.device)
    scoring_ref.check_logprobs([None if g is None else g[at] for g in got], x[at], t[at], top)


@pytest.mark.parametrize("dtype,rows,v,pad", [("bf16", 8192, 8195, 0), ("bf16", 2730, 49153, 0), ("bf16", 2047, 65537, 0),
                                              ("fp32", 4096, 4097, 0), ("bf16", 4096, 16390, 1), ("bf16", 3000, 8200, 1),
                                              ("fp32", 620, 49155, 0), ("bf16", 1500, 8192, 3)])
@pytest.mark.parametrize("top", [0, 5, 64])
def test_rows_that_end_just_past_a_tile(lib, dtype, rows, v, pad, top):
    """Rows whose last tile holds no whole vector, or none at some starts in memory; several rows to a CTA."""
    from minitp_b200 import ops

    r = torch.Generator(device="cuda").manual_seed(rows + v)
    wide = torch.empty(rows, v + pad, dtype=DT[dtype], device="cuda")
    wide.normal_(0.0, 3.0, generator=r)
    x = wide[:, pad:]
    t = torch.randint(0, v, (rows,), generator=r, device="cuda")
    t[::3] = v - 1
    x[::4, -1] = 20.0  # the best, outside the whole vectors
    _check_some(ops.token_logprobs(x, t, top), x, t, top)
    _status_is_clean(lib)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("top", [0, 5, 64])
def test_shards_of_fewer_tiles_than_planned(lib, dtype, top):
    """Shards of no, few and most of the planned columns, with many rows to a CTA."""
    from minitp_b200 import ops

    rows, plan, cuts = 4096, 20000, [0, 9000, 9000, 17200, 17203]
    r = torch.Generator(device="cuda").manual_seed(top)
    x = torch.empty(rows, cuts[-1], dtype=DT[dtype], device="cuda").normal_(0.0, 3.0, generator=r)
    t = torch.randint(0, cuts[-1], (rows,), generator=r, device="cuda")
    blocks = [ops.logprobs_block(x[:, a:b], t, top, a, plan) for a, b in zip(cuts, cuts[1:])]
    _check_some(ops.logprobs_join(torch.stack(blocks), t, (rows,), top, plan, DT[dtype]), x, t, top, 41)
    _status_is_clean(lib)
