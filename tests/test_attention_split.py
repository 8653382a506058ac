"""How the attention over listed blocks cuts its work into thread blocks' shares, replayed on the host from the header that the kernel is
built from: every slice once and every part joined for lists that ascend; nothing outside the arrays and the workspace for any others."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
LEAD = {False: 16, True: 24}


@pytest.fixture(scope="module")
def replay(tmp_path_factory):
    cxx = os.environ.get("CXX") or shutil.which("g++") or shutil.which("c++")
    if not cxx:
        pytest.skip("no C++ compiler")
    so = str(tmp_path_factory.mktemp("split") / "split_replay.so")
    src = os.path.join(os.path.dirname(HERE), "unified-cache-management_b200", "csrc")
    subprocess.run([cxx, "-O1", "-std=c++17", "-Wall", "-fPIC", "-shared", "-I", src,
                    os.path.join(HERE, "split_replay.cpp"), "-o", so], check=True)
    lib = C.CDLL(so)
    lib.replay.restype = C.c_int64

    def run(offsets, total, spe, heads, blocks, tiles=None, tiled=False):
        off = np.asarray(offsets, np.int32)
        n_req = len(off) - 1
        t = None if tiles is None else np.asarray(tiles, np.int32)
        col = 1 if t is None else int(t.max())
        room = 8 * (n_req + 1) * heads * col + 8 * blocks
        out = np.zeros((room, 10), np.int64)
        rejected, reported = C.c_int64(), C.c_int32()
        p = lambda a, ty: None if a is None else a.ctypes.data_as(C.POINTER(ty))  # noqa: E731
        n = lib.replay(p(off, C.c_int32), n_req, total, spe, heads, p(t, C.c_int32), col, LEAD[tiled or t is not None], blocks,
                       p(out, C.c_int64), C.c_int64(room), C.byref(rejected), C.byref(reported))
        assert n != -2, "a batch that the host refuses"
        assert n >= 0, "a loop that does not end"
        rows = out[:n]
        block, r, h, ct, lo, hi, first, entries, begins, parts = rows.T
        # nothing outside: lists, heads, slices, and the parts that the joining kernel would read
        assert bool(((r >= 0) & (r < max(n_req, 1)) & (h >= 0) & (h < heads) & (ct >= 0)).all())
        assert bool(((first >= 0) & (entries >= 0) & (first + entries <= total)).all())
        assert bool(((lo >= 0) & (hi <= entries * spe)).all())
        assert bool(((parts >= 0) & (block + parts <= blocks)).all()), "more parts than thread blocks"
        return rows, rejected.value, bool(reported.value)

    run.lib = lib
    return run


def check_cover(rows, offsets, spe, heads, tiles):
    """Every slice of every item once; the parts of a split item in neighbouring thread blocks, the first of them says how many."""
    items = {}
    for block, r, h, ct, lo, hi, first, entries, begins, parts in rows.tolist():
        assert first == offsets[r] and entries == offsets[r + 1] - offsets[r]
        items.setdefault((r, h, ct), []).append((block, lo, hi, begins, parts))
    want = {(r, h, ct) for r in range(len(offsets) - 1) for h in range(heads) for ct in range(tiles[r])}
    assert set(items) == want
    for (r, _, _), segs in items.items():
        segs.sort()
        n = (offsets[r + 1] - offsets[r]) * spe
        assert segs[0][1] == 0 and segs[-1][2] == n
        assert all(a[2] == b[1] and a[0] + 1 == b[0] for a, b in zip(segs, segs[1:]))
        assert segs[0][3] == 1 and not any(s[3] for s in segs[1:])
        assert segs[0][4] == (len(segs) if len(segs) > 1 else 0) and not any(s[4] for s in segs[1:])


@pytest.mark.parametrize("seed", range(40))
def test_every_slice_once_and_every_part_joined(replay, seed):
    rng = np.random.default_rng(seed)
    for _ in range(12):
        n_req = int(rng.choice([1, 2, 3, 20, 31, 32, 63, 200, 1100]))
        most = int(rng.choice([1, 4, 40, 900])) if n_req < 200 else 6
        counts = rng.integers(0, most + 1, n_req)
        start = int(rng.integers(0, 5))
        off = (start + np.concatenate([[0], np.cumsum(counts)])).tolist()
        total = off[-1] + int(rng.integers(0, 9))
        spe, heads, blocks = int(rng.choice([1, 2, 8])), int(rng.choice([1, 2, 8])), int(rng.choice([1, 7, 148, 592]))
        if n_req > 1000:
            heads = 1
        tiled = bool(rng.integers(0, 2))
        tiles = rng.integers(1, 4, n_req) if tiled and n_req <= 1023 and rng.integers(0, 2) else None
        rows, rejected, reported = replay(off, total, spe, heads, blocks, tiles, tiled)
        assert rejected == 0 and not reported
        check_cover(rows, off, spe, heads, [1] * n_req if tiles is None else tiles.tolist())


BROKEN = [
    # offsets, entries, slices per block, heads
    ([0, 100_000, 10], 100_000, 1, 1),
    ([0, 100_000, 1], 100_000, 1, 2),
    ([0, 1000, 600], 1000, 8, 8),
    ([0, 108, 1], 108, 1, 2),
    ([0, 6, 3, 90, 40], 108, 1, 2),
    ([50, 40, 30, 20, 10], 108, 4, 1),
    ([0, 2_000_000_000, -5, 7, 108], 108, 1, 2),
    ([0, 6, 200, 100, 108], 108, 1, 2),
    ([0, 5, 109], 108, 1, 1),
    ([-1, 5, 108], 108, 1, 1),
    ([40, 0, 40, 0, 40, 108], 108, 2, 8),
    ([2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1], 50, 1, 1),
]


@pytest.mark.parametrize("off,total,spe,heads", BROKEN)
@pytest.mark.parametrize("tiles", [None, 1, 3])
def test_offsets_that_lists_cannot_have_reach_nothing_outside(replay, off, total, spe, heads, tiles):
    for blocks in (1, 22, 148, 592):
        t = None if tiles is None else [1 + (i + tiles) % 3 for i in range(len(off) - 1)]
        _, _, reported = replay(off, total, spe, heads, blocks, t)
        assert reported


def test_zigzag_offsets_that_add_up_to_more_than_there_are_units(replay):
    """Up and down again through all entries, so often that the sum over the requests passes 2^31."""
    n = 1000
    off = [0 if i % 2 else 1_000_000 for i in range(n + 1)]
    for heads, total in ((1, 2_000_000), (8, 1_000_000), (1, 300_000_000)):
        off = [0 if i % 2 else total for i in range(n + 1)]
        for tiles in ([1 + i % 3 for i in range(n)], [3] * n, None):
            if tiles is not None and total > 10 ** 8:
                tiles = [1 + i % 2 for i in range(n)]
            _, _, reported = replay(off, total, 1, heads, 592, tiles)
            assert reported


@pytest.mark.parametrize("seed", range(30))
def test_any_offsets_at_all(replay, seed):
    rng = np.random.default_rng(1000 + seed)
    for _ in range(30):
        n_req = int(rng.choice([1, 2, 5, 31, 40, 500, 1023]))
        total = int(rng.choice([1, 50, 3000, 1_000_000]))
        lo, hi = [(0, total), (-total, 2 * total), (-2 ** 31, 2 ** 31 - 1)][int(rng.integers(0, 3))]
        off = rng.integers(lo, hi, n_req + 1, endpoint=True)
        if rng.integers(0, 2):                                            # mostly ascending, a few that are not
            off = np.sort(off)
            for i in rng.integers(0, n_req + 1, 2):
                off[i] = rng.integers(lo, hi, endpoint=True)
        spe, heads = int(rng.choice([1, 8])), int(rng.choice([1, 8]))
        tiles = rng.integers(0, 4, n_req) if rng.integers(0, 2) else None
        if tiles is not None:
            tiles[0] = max(tiles[0], 1)
        _, _, reported = replay(off, total, spe, heads, int(rng.choice([1, 22, 592])), tiles)
        off = off.astype(np.int64)
        assert reported == bool((off < 0).any() or (off > total).any() or (np.diff(off) < 0).any())


def test_places_in_a_row_of_a_block_table(replay):
    """A place is looked up where it lies inside its row and inside the table, whatever the row's offsets are: no difference of them wraps."""
    ends = [-2 ** 31, -2 ** 31 + 1, -7, -1, 0, 1, 5, 6, 90, 100, 101, 2 ** 30, 2 ** 31 - 2, 2 ** 31 - 1]
    for t0 in ends:
        for t1 in ends:
            for size in (0, 1, 100, 2 ** 31 - 1):
                for at in (0, 1, 4, 94, 99, 100, 2 ** 31 - 1):
                    want = t0 >= 0 and t0 + at < min(t1, size)
                    assert replay.lib.row_holds(t0, t1, size, at) == want, (t0, t1, size, at)
