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
