"""Replay of the log-probability kernel's waits on the host: no CTA comes to a stop, and the plan covers every tile."""

import ctypes
import itertools
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
TILE = {2: 8192, 4: 4096}  # columns, by the element's bytes


@pytest.fixture(scope="module")
def replay(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("schedule") / "schedule.so")
    csrc = os.path.join(os.path.dirname(HERE), "minitp_b200", "csrc")
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I", csrc, "-x", "c++",
                    os.path.join(HERE, "logprobs_schedule.cpp"), "-o", so], check=True)
    lib = ctypes.CDLL(so)
    lib.lp_blocked.argtypes = [ctypes.c_longlong, ctypes.c_int, ctypes.c_int, ctypes.c_longlong] + [ctypes.c_int] * 4 + \
        [ctypes.POINTER(ctypes.c_int)] * 2
    lib.lp_plan_wrong.argtypes = [ctypes.c_longlong, ctypes.c_int, ctypes.c_int]

    def blocked(rows, v, plan=None, ld=None, base=0, es=2, k=5, skip=False):
        ctas, run = ctypes.c_int(), ctypes.c_int()
        n = lib.lp_blocked(rows, v, plan or v, ld or v, base, es, k, int(skip), ctypes.byref(ctas), ctypes.byref(run))
        return n, ctas.value, run.value

    blocked.lib = lib
    return blocked


def test_a_copy_that_passes_over_empty_tiles_would_block(replay):
    """The replay tells a schedule that stops from one that does not."""
    for case in (dict(rows=8192, v=8195), dict(rows=4096, v=4097, es=4), dict(rows=4096, v=16390, ld=16391),
                 dict(rows=4096, v=9000, plan=20000), dict(rows=2730, v=49153), dict(rows=2047, v=65537)):
        blocked, ctas, _ = replay(**case, skip=True)
        assert blocked >= ctas - 1 > 400
        assert replay(**case)[0] == 0
    assert replay(512, 152064, k=20, skip=True)[0] == 0  # (no empty tile)


@pytest.mark.parametrize("es", [2, 4])
@pytest.mark.parametrize("tiles", [1, 2, 6])
def test_no_cta_stops(replay, es, tiles):
    """Vocabularies from a tile's end on, rows at every start in memory, and 1 to 40 tiles a CTA."""
    ve = 16 // es
    for over, k, (rows, pad), base in itertools.product(range(16), (0, 1, 5, 33, 64),
                                                        ((1, 0), (444, 1), (3001, ve - 1), (17000, 0)), (0, es, 16 - es)):
        v = tiles * TILE[es] + over
        blocked, _, run = replay(rows // tiles + 1, v, ld=v + pad, base=base, es=es, k=k)
        assert blocked == 0, (v, k, rows, pad, base, run)


@pytest.mark.parametrize("es", [2, 4])
def test_no_cta_stops_on_a_shard_of_fewer_columns(replay, es):
    plan = 5 * TILE[es] // 2
    for v, k, rows in itertools.product((0, 1, 7, TILE[es] - 1, TILE[es], TILE[es] + 3, 2 * TILE[es] + 1, plan), (0, 1, 5, 64),
                                        (1, 300, 4096)):
        assert replay(rows, v, plan, ld=max(v, 1) + 1, es=es, k=k)[0] == 0, (v, k, rows)


def test_the_plan_covers_every_tile(replay):
    for rows, v, es in itertools.product((1, 2, 147, 444, 445, 3000, 20000), (1, 8192, 8193, 40000, 151936, 10 ** 6), (2, 4)):
        assert replay.lib.lp_plan_wrong(rows, v, es) == 0, (rows, v, es)
    assert replay.lib.lp_plan_wrong(1, 2 ** 30 - 1, 2) == 0
