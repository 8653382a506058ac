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
    """The same queries again: every block is resident, none but the newest ones may move, and each layer reads its own blocks."""
    eng = make()
    eng.make_queries()
    for _ in range(3):
        eng.step()
        check(eng)
    newest = set(eng.new_block_ids.tolist())
    table, boff, off = eng.block_table.tolist(), eng.offsets.tolist(), eng.k_offsets.tolist()
    for l in range(eng.L):
        for r in range(eng.batch.n_req):
            moved = eng.remap_out[l][1][off[r]:off[r + 1]].tolist()
            assert all(table[boff[r] + x] in newest for x in moved if x >= 0)
    a, b = (set(eng.sel_ids[l].tolist()) for l in (0, 1))
    assert a != b                                   # (the layers do select different blocks)


@pytest.mark.parametrize("kw", [{}, dict(overlap=True)])
def test_newly_selected_blocks_are_all_loaded(kw):
    """Queries that drift: some of each selection is resident, the rest is moved, and none of it is left out."""
    eng = make(n_layers=3, **kw)
    eng.make_queries()
    eng.step()
    check(eng)
    for _ in range(4):
        eng.drift_queries(0.7)
        eng.step()
        check(eng)
        assert 0 < eng.loads_of_last_step() < eng.L * eng.batch.total_k
        for l in range(eng.L):
            n = eng.sel_counts[l].tolist()
            off = eng.k_offsets.tolist()
            served = torch.cat([eng.remap_out[l][0][off[r]:off[r] + n[r]] for r in range(eng.batch.n_req)])
            assert bool((served >= 0).all())
    eng.capture()
    for _ in range(3):
        eng.drift_queries(0.7)
        eng.step()
        check(eng)


@pytest.mark.parametrize("kw", [{}, dict(overlap=True)])
def test_a_block_that_filled_up_is_moved_again(kw):
    """Every block is selected and resident; the newest one of each request changes in the pool between the steps."""
    eng = make(ratio=1.0, **kw)
    eng.make_queries()
    eng.step()
    check(eng)
    new = eng.new_block_ids.long()

    def refill():
        eng.kv_pool[:, new] = torch.randn(eng.kv_pool[:, new].shape, device=DEV, generator=eng.gen).to(torch.bfloat16)

    refill()
    eng.step()
    check(eng)
    assert eng.loads_of_last_step() == eng.L * eng.batch.n_req      # the newest blocks and no others
    eng.capture()
    refill()
    eng.step()
    check(eng)


@pytest.mark.parametrize("kw", [dict(cache_bits=4), dict(delta=True)])
def test_representatives_of_the_whole_pool_renew_what_the_attention_reads(kw):
    """prefill_pool_all says that the pool holds new blocks: the quantised copy and the working sets hold them then, too."""
    from test_gpu_engine_attention import make as make_any
    eng = make_any(**kw)
    eng.make_queries()
    eng.step()
    check(eng, kw.get("cache_bits", 16))
    eng.kv_pool.copy_(torch.randn(eng.kv_pool.shape, device=DEV, generator=eng.gen).to(torch.bfloat16))
    for l in range(eng.L):
        eng.prefill_pool_all(l)
    eng.step()
    check(eng, kw.get("cache_bits", 16))


@pytest.mark.parametrize("kw", [dict(cache_bits=8), dict(delta=True)])
def test_pooling_a_layer_renews_what_its_attention_reads(kw):
    """pool_layer, in place of the pooling that a step begins with, says the same of the newest blocks."""
    from test_gpu_engine_attention import make as make_any
    eng = make_any(**kw)
    eng.make_queries()
    eng.step()
    new = eng.new_block_ids.long()
    eng.kv_pool[:, new] = torch.randn(eng.kv_pool[:, new].shape, device=DEV, generator=eng.gen).to(torch.bfloat16)
    for l in range(eng.L):
        eng.pool_layer(l)
        eng.layer_step(l)
    check(eng, kw.get("cache_bits", 16))


def test_remap_without_a_deferred_free_list():
    """slot_free None: with as many slots as selected blocks every block is served in every round, hits stay, slots are distinct."""
    import numpy as np
    from ucmx import ops
    rng = np.random.default_rng(7)
    n_logical, ks = [300, 64, 9], [40, 64, 3]
    off = np.concatenate([[0], np.cumsum(ks)]).astype(np.int32)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)  # noqa: E731
    logical, phys = t(np.full(107, -1)), t(np.arange(107))
    resident = {}
    for _ in range(5):
        sel = np.concatenate([np.sort(rng.choice(n, k, replace=False)) for n, k in zip(n_logical, ks)]).astype(np.int32)
        table, ll, lp, lc = ops.remap_resident(logical, None, phys, t(off), t(sel), t(off), max_logical=300, max_slots=64)
        table, lc = table.cpu().numpy(), lc.cpu().numpy()
        new = {}
        for r in range(3):
            a, b = off[r], off[r + 1]
            assert sorted(table[a:b]) == list(range(a, b))                   # every slot of the request serves one block
            assert lc[r] == sum((r, int(x)) not in resident for x in sel[a:b])
            for x, s in zip(sel[a:b], table[a:b]):
                assert resident.get((r, int(x)), s) == s
                new[r, int(x)] = s
        resident = new


@pytest.mark.parametrize("overlap", [False, True])
def test_the_delta_step_alone_serves_its_whole_selection(overlap):
    """Without an attention behind it, too: each selected block has a slot, and what is loaded is what was not resident."""
    from ucmx.engine import DecodeRetrievalEngine
    from ucmx.workloads import KvShape, ragged_decode_batch
    shape = KvShape(n_q_heads=8, n_kv_heads=2, head_dim=128, block_tokens=64, n_layers=2)
    batch = ragged_decode_batch(seed=44, n_req=6, min_ctx=512, max_ctx=4096, block_tokens=64, ratio=0.3, min_k=3)
    eng = DecodeRetrievalEngine(shape, batch, DEV, seed=6, delta=True, overlap=overlap)
    eng.make_queries()
    off, newest = eng.k_offsets.tolist(), (eng.offsets[1:] - eng.offsets[:-1] - 1).tolist()
    before = [[set() for _ in range(6)] for _ in range(2)]
    for step in range(5):
        eng.step()
        for l in range(2):
            table, sel, n = eng.remap_out[l][0].tolist(), eng.sel_ids[l].tolist(), eng.sel_counts[l].tolist()
            for r in range(6):
                a, b = off[r], off[r] + n[r]
                assert sorted(table[a:b]) == list(range(a, b))            # (k is the number of slots)
                resident = before[l][r] - {newest[r]}
                assert int(eng.remap_out[l][3][r]) == len(set(sel[a:b]) - resident)
                before[l][r] = set(sel[a:b])
        eng.drift_queries(0.6)


@pytest.mark.parametrize("overlap", [False, True])
def test_delta_steps_with_host_buffers_attend_to_their_selection(overlap):
    """The end-to-end step, launched and from its graph: queries and a refilled block new each time."""
    eng = make(overlap=overlap)
    eng.make_queries()
    eng.alloc_host()
    new = eng.new_block_ids.long()
    for step in range(5):
        if step == 2:
            eng.capture_host()
        eng.kv_pool[:, new] = torch.randn(eng.kv_pool[:, new].shape, device=DEV, generator=eng.gen).to(torch.bfloat16)
        noise = torch.randn(eng.q_host.shape, generator=torch.Generator().manual_seed(step))
        eng.q_host.copy_((0.7 * eng.q_host.float() + 0.7 * noise).to(torch.bfloat16))
        torch.cuda.synchronize()
        eng.step_host()
        check(eng)
