"""The finder of prompt attention's tiles on the host: every token in one tile, and nothing outside the queries."""

import bisect
import ctypes
import os
import random
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("tiles") / "tiles.so")
    csrc = os.path.join(os.path.dirname(HERE), "minitp_b200", "csrc")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", csrc, "-I", HERE, "-x", "c++",
                    os.path.join(HERE, "prompt_tiles.cpp"), "-o", so], check=True)
    return ctypes.CDLL(so)


def _ints(values):
    return (ctypes.c_int * max(1, len(values)))(*values)


def _find(host, starts, first, n, total, hq, hkv, rows, numbers, name="pt_find"):
    """([(start, tok0, ntok)], tokens a tile, planned items, (gap0, gap1))"""
    out, tt, items, gaps = _ints([0] * (3 * len(numbers))), ctypes.c_int(), ctypes.c_longlong(), _ints([0, 0])
    apart = getattr(host, name)(_ints(starts), len(starts) - 1, first, n, total, hq, hkv, rows, _ints(numbers), len(numbers),
                                out, ctypes.byref(tt), ctypes.byref(items), gaps)
    assert apart == 0
    return [tuple(out[3 * i:3 * i + 3]) for i in range(len(numbers))], tt.value, items.value, (gaps[0], gaps[1])


def _starts(r, count, longest, at=0):
    out = [at]
    for _ in range(count):
        out.append(out[-1] + (0 if r.random() < 0.2 else r.randint(1, longest)))
    return out


def _check(tiles, tt, starts, first, n):
    """Every token of a prompt among the queries lies in one tile, with its prompt's start."""
    want = {}
    for a, b in zip(starts, starts[1:]):
        for tok in range(max(a, first), min(b, first + n)):
            want[tok] = a
    got = {}
    for start, tok0, ntok in tiles:
        assert 0 <= ntok <= tt
        for tok in range(tok0, tok0 + ntok):
            assert tok not in got
            got[tok] = start
    assert got == want


COUNTS = [0, 1, 2, 31, 32, 33, 63, 64, 65, 96, 97, 128, 129, 300]


@pytest.mark.parametrize("count", COUNTS)
def test_every_token_is_in_one_tile(host, count):
    r = random.Random(count)
    for hq, hkv, rows, longest in [(4, 2, 16, 9), (14, 2, 128, 40), (28, 4, 256, 90), (7, 1, 64, 3), (300, 1, 128, 4)]:
        starts = _starts(r, count, longest, at=r.randint(0, 5))
        total = starts[-1] + r.randint(0, 7)
        for first, n in [(0, total), (total // 3, total - total // 3), (total // 4, total // 2)]:
            if n == 0:
                continue
            tt = _find(host, starts, first, n, total, hq, hkv, rows, [])[1]
            tiles, tt, items, gaps = _find(host, starts, first, n, total, hq, hkv, rows, list(range(n // tt + count + 1)))
            assert items % (n // tt + count) == 0 if n // tt + count else items == 0
            assert tiles[-1][2] == 0  # no tile behind those planned for
            _check(tiles, tt, starts, first, n)
            assert gaps == (min(max(starts[0], first), first + n), min(max(starts[-1], first), first + n))


@pytest.mark.parametrize("count", [1, 64, 65, 200])
def test_starts_in_disorder_stay_within_the_tokens(host, count):
    r = random.Random(count)
    for _ in range(20):
        total = r.randint(1, 400)
        starts = [r.choice([r.randint(-50, total + 50), -2 ** 31, 2 ** 31 - 1]) for _ in range(count + 1)]
        first = r.randint(0, total - 1)
        n = r.randint(1, total - first)
        tiles, tt, _, gaps = _find(host, starts, first, n, total, 4, 2, 16, list(range(n + count + 1)))
        seen = set()
        for start, tok0, ntok in tiles:
            if ntok:
                assert first <= tok0 and tok0 + ntok <= first + n and 0 <= start <= tok0
                assert seen.isdisjoint(range(tok0, tok0 + ntok))
                seen.update(range(tok0, tok0 + ntok))
        assert all(first <= g <= first + n for g in gaps)


@pytest.mark.parametrize("count", [3, 64, 65, 300])
def test_a_finder_left_early_leaves_gaps_within_the_tokens(host, count):
    """Whoever stops after a wait that ran out, with prompts still unread, zeroes no rows outside the output."""
    starts = _starts(random.Random(count), count, 9, at=4)
    total = starts[-1] + 3
    for numbers in ([], [0], [0, 1, 2]):
        _, _, _, gaps = _find(host, starts, 2, total - 2, total, 4, 2, 16, numbers)
        assert gaps[0] == 4 and 2 <= gaps[1] <= total
        assert gaps[1] in (starts[-1], total)  # the last prompt's end, or (not read yet) nothing to zero


@pytest.mark.parametrize("count", COUNTS)
def test_a_tile_found_by_itself(host, count):
    """Each number on its own, as a CTA with one tile asks for it: every token in one tile, planned numbers only."""
    r = random.Random(count + 7)
    for hq, hkv, rows, longest in [(4, 2, 16, 9), (8, 4, 32, 20), (300, 1, 16, 4)]:
        starts = _starts(r, count, longest, at=r.randint(0, 5))
        total = starts[-1] + r.randint(0, 7)
        for first, n in [(0, total), (total // 3, total - total // 3), (total // 4, total // 2)]:
            if n == 0:
                continue
            tt = _find(host, starts, first, n, total, hq, hkv, rows, [])[1]
            numbers = list(range(n // tt + count + 1))
            tiles, _, _, gaps = _find(host, starts, first, n, total, hq, hkv, rows, numbers, "pt_only")
            assert tiles[-1][2] == 0
            _check(tiles, tt, starts, first, n)
            assert gaps == (min(max(starts[0], first), first + n), min(max(starts[-1], first), first + n))


def test_a_tile_among_a_million_prompts(host):
    r = random.Random(3)
    starts = _starts(r, 1 << 20, 3)
    total = starts[-1]
    for first, n in [(0, total), (1000, total - 2000)]:
        tt = _find(host, starts, first, n, total, 4, 2, 16, [0], "pt_only")[1]
        numbers = sorted(r.randrange(n // tt + (1 << 20)) for _ in range(1500))
        tiles, _, _, _ = _find(host, starts, first, n, total, 4, 2, 16, numbers, "pt_only")
        at = {}
        for start, tok0, ntok in tiles:
            if ntok:
                at[tok0] = start
        for tok0, start in at.items():
            s = bisect.bisect_right(starts, tok0) - 1
            assert starts[s] == start and first <= tok0 < first + n
        assert len(at) > 500


def test_a_tile_by_itself_of_starts_in_disorder(host):
    r = random.Random(9)
    for count in (65, 200, 1000):
        for _ in range(10):
            total = r.randint(1, 400)
            starts = [r.choice([r.randint(-50, total + 50), -2 ** 31, 2 ** 31 - 1]) for _ in range(count + 1)]
            first = r.randint(0, total - 1)
            n = r.randint(1, total - first)
            tiles, _, _, gaps = _find(host, starts, first, n, total, 4, 2, 16, list(range(n + count + 1)), "pt_only")
            assert all(first <= tok0 and tok0 + ntok <= first + n and 0 <= start <= tok0 for start, tok0, ntok in tiles if ntok)
            assert all(first <= g <= first + n for g in gaps)
