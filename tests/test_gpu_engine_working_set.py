"""The delta step's attention reads a resident working set: what it reads must be the blocks that the layer selected, as they are in
the pool now, in every step and not the first alone."""
import pytest
import torch

from test_gpu_engine_attention import DEV, check

pytestmark = pytest.mark.gpu


def make(ratio=0.2, n_layers=2, **kw):
    from ucmx.engine import DecodeRetrievalEngine
    from ucmx.workloads import KvShape, ragged_decode_batch
    shape = KvShape(n_q_heads=8, n_kv_heads=2, head_dim=128, block_tokens=64, n_layers=n_layers)
    batch = ragged_decode_batch(seed=43, n_req=5, min_ctx=512, max_ctx=4096, block_tokens=64, ratio=ratio, min_k=3)
    return DecodeRetrievalEngine(shape, batch, DEV, with_kv_pool=True, seed=5, attend=True, delta=True, **kw)


def test_every_layer_keeps_a_working_set_of_its_own():
    """The same queries again: every block is resident, nothing moves, and each layer reads its own blocks."""
    eng = make()
    eng.make_queries()
    for _ in range(3):
        eng.step()
        check(eng)
    assert eng.loads_of_last_step() == 0
    a, b = (set(eng.sel_ids[l].tolist()) for l in (0, 1))
    assert a != b                                   # (the layers do select different blocks)
