"""Attention over listed blocks: what the header allows of a workspace."""
import pytest
import torch

import attention_ref as R
from test_gpu_block_attention import DEV, Setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", [16, 8, 4])
@pytest.mark.parametrize("H,G,D,T,counts,nq", [
    (2, 4, 128, 16, [300, 2, 500], None), (1, 1, 64, 16, [800], None), (1, 8, 256, 16, [300], None), (2, 12, 64, 16, [200, 90], [2, 1]),
])
def test_a_workspace_that_starts_on_16_bytes_and_no_more(fmt, H, G, D, T, counts, nq):
    from ucmx import ops
    s = Setup(90, fmt, H, G, D, T, counts, nq).tails()
    need = ops.attention_workspace(s.q.to(DEV), H, max_q_tokens=max(s.nq), bits=fmt).numel()
    room = torch.full((need + 64,), 255, dtype=torch.uint8, device=DEV)
    ws = room[16:16 + need]
    assert ws.data_ptr() % 32 == 16
    out, _, tol, _ = s.want()
    R.check(s.run(workspace=ws), out, tol)
    assert bool((room[:16] == 255).all()) and bool((room[16 + need:] == 255).all())      # nothing beside it is written


@pytest.mark.parametrize("fmt,nq", [(16, 1), (16, 5), (4, 1), (8, 3)])
def test_every_call_with_offsets_that_lists_cannot_have_says_so(fmt, nq):
    """Each of them by itself; nothing beside the workspace and out is written, and the next call is fine."""
    from ucmx import _native, ops
    s = Setup(91, fmt, 2, 8, 64, 16, [6, 90, 4, 8], [nq] * 4).tails()
    need = ops.attention_workspace(s.q.to(DEV), 2, max_q_tokens=nq, bits=fmt).numel()
    room = torch.full((need + (1 << 20),), 255, dtype=torch.uint8, device=DEV)
    _native.device_error()
    for off in ([0, 108, 1, 108, 108], [0, 1, 108, 1, 1], [0, 6, 3, 90, 40], [0, 108, 0, 108, 0], [50, 40, 30, 20, 10], [0, 2_000_000_000, -5, 7, 108],
                [0, 6, 200, 100, 108], [0, 6, 96, 100, 109], [-1, 6, 96, 100, 108], [108, 0, 0, 0, 0]):
        s.run(offsets=torch.tensor(off, dtype=torch.int32, device=DEV), workspace=room[:need])
        torch.cuda.synchronize()
        assert _native.device_error() == 3, off
        assert bool((room[need:] == 255).all())
    s.run(offsets=torch.tensor([3, 9, 9, 60, 108], dtype=torch.int32, device=DEV), workspace=room[:need])
    torch.cuda.synchronize()
    assert _native.device_error() == 0
    s.check()


@pytest.mark.parametrize("fmt,G", [(16, 16), (16, 1), (4, 8)])
def test_query_offsets_that_batches_cannot_have_are_reported_wherever_they_stand(fmt, G):
    """A request whose query tokens go backwards, are more than the call allows or lie outside the queries: code 3, whichever request it is."""
    from ucmx import _native
    n = 40
    s = Setup(92, fmt, 2, G, 64, 16, [3] * n, [3] * n).tails()
    good = s.qoff.tolist()
    _native.device_error()
    for at, value in ((1, -1), (9, 0), (20, 80), (33, 10), (39, 113), (40, 121), (40, 2 ** 31 - 1), (17, -2 ** 31), (40, 100), (40, -5), (0, -3)):
        off = list(good)
        off[at] = value
        s.run(q_offsets=torch.tensor(off, dtype=torch.int32, device=DEV))
        torch.cuda.synchronize()
        assert _native.device_error() == 3, (at, value)
    s.check()


def test_rows_of_a_block_table_that_begin_or_end_anywhere():
    """Table offsets beyond the table, backwards and at the ends of their type: the entries are dropped and reported."""
    import numpy as np
    from ucmx import _native
    for fmt in (16, 4):
        s = Setup(93, fmt, 2, 4, 128, 16, [6, 5])
        table = s.ids.copy()
        s.positions = np.asarray([5, 0, 2, 4, 1, 3, 0, 4, 2, 1, 3], np.int32)
        for off, held in (([0, 6, 11], (6, 5)), ([0, 5, -2 ** 31], (5, 0)), ([-2 ** 31, 6, 11], (0, 5)), ([2 ** 31 - 1, 6, 2 ** 31 - 1], (0, 5)),
                          ([3, 2, 4], (0, 2)), ([-1, 6, 9], (0, 3))):
            row = [(off[0], held[0]), (off[1], held[1])]
            s.ids = np.asarray([table[row[i // 6][0] + p] if p < row[i // 6][1] else -1 for i, p in enumerate(s.positions)], np.int32)
            want = s.want()
            _native.device_error()
            got = s.run(block_ids=None, block_table=torch.from_numpy(table).to(DEV), table_offsets=torch.tensor(off, dtype=torch.int32, device=DEV))
            torch.cuda.synchronize()
            assert _native.device_error() == (0 if held == (6, 5) else 3), off
            R.check(got, want[0], want[2], str(off))
