"""The decode step that ends in attention: the engine's output per layer is the attention over the blocks that it selected, whichever
way the step runs, over the bf16 pool, the resident working set of the delta step and quantised copies of the pool."""
import pytest
import torch

import attention_ref as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def make(**kw):
    from ucmx.engine import DecodeRetrievalEngine
    from ucmx.workloads import KvShape, ragged_decode_batch
    shape = KvShape(n_q_heads=8, n_kv_heads=2, head_dim=128, block_tokens=64, n_layers=2)
    batch = ragged_decode_batch(seed=41, n_req=5, min_ctx=512, max_ctx=4096, block_tokens=64, ratio=0.2, min_k=3)
    return DecodeRetrievalEngine(shape, batch, DEV, with_kv_pool=True, seed=3, attend=True, **kw)


def check(eng, bits=16):
    torch.cuda.synchronize()
    from ucmx import _native
    assert _native.device_error() == 0
    off, cnt = eng.k_offsets.cpu().tolist(), eng.sel_counts.cpu()
    if bits == 16:
        k, v, err = eng.kv_pool[0].cpu().double(), eng.kv_pool[1].cpu().double(), 0.0
    else:
        k, v = R.values(R.pack(eng.kv_pool[0].cpu(), eng.kv_pool[1].cpu(), bits), eng.D, bits)
        err = 12.0
    table, boff = eng.block_table.cpu(), eng.offsets.cpu().tolist()
    for l in range(eng.L):
        sel = eng.sel_ids[l].cpu()
        lists = []
        for r in range(eng.batch.n_req):
            ids = sel[off[r]:off[r] + int(cnt[l, r])].tolist()
            if eng.delta:
                ids = [int(table[boff[r] + i]) for i in ids]
            lists.append((range(r, r + 1), [(int(b), i) for i, b in enumerate(ids)], None))
        out, _, tol, _ = R.attend(eng.q_dev[l].cpu(), k, v, lists, codes_err=err)
        R.check(eng.attn_out[l], out, tol, f"layer {l}")


@pytest.mark.parametrize("kw,bits", [({}, 16), (dict(cache_bits=4), 4), (dict(cache_bits=8), 8), (dict(delta=True), 16),
                                     (dict(overlap=True), 16), (dict(overlap=True, cache_bits=4), 4)])
def test_attention_at_the_end_of_the_step(kw, bits):
    eng = make(**kw)
    eng.make_queries()
    eng.step()
    check(eng, bits)
    # a block fills up between the steps, queries move on; then the same from a captured graph
    new = eng.new_block_ids.long()
    eng.kv_pool[:, new] = torch.randn(eng.kv_pool[:, new].shape, device=DEV, generator=eng.gen).to(torch.bfloat16)
    eng.drift_queries(0.5)
    if not eng.delta:
        eng.step()
        check(eng, bits)
        eng.capture()
        eng.drift_queries(0.5)
    eng.step()
    if not eng.delta:
        check(eng, bits)


def test_steps_with_host_buffers_attend_too():
    eng = make()
    eng.make_queries()
    eng.alloc_host()
    eng.step_host()
    check(eng)
    eng.capture_host()
    eng.q_host.copy_(torch.randn(eng.q_host.shape).to(torch.bfloat16))
    eng.step_host()
    check(eng)


def test_refusals():
    with pytest.raises(ValueError):
        make(delta=True, cache_bits=4)
    from ucmx.engine import DecodeRetrievalEngine
    from ucmx.workloads import KvShape, fixed_batch
    with pytest.raises(ValueError):
        DecodeRetrievalEngine(KvShape(n_layers=1), fixed_batch(1, 2, 1), DEV, with_kv_pool=False, attend=True)
    with pytest.raises(ValueError):
        DecodeRetrievalEngine(KvShape(n_layers=1), fixed_batch(1, 2, 1), DEV, cache_bits=4)
