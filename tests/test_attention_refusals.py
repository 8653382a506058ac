"""What the quantised cache and the attention over listed blocks refuse before anything is launched (no GPU needed)."""
import ctypes as C

import pytest
import torch

import attention_ref as R

FAKE = 0x10000           # an address that is never used: every call here is refused on the host


def geom(**kw):
    from ucmx import _native as N
    a = dict(block_stride=16 * 2 * 128, token_stride=2 * 128, block_tokens=16, n_kv_heads=2, head_dim=128, reserved=4)
    a.update(kw)
    return C.byref(N.KvGeometry(*a.values()))


def qgeom(**kw):
    from ucmx import _native as N
    a = dict(n_blocks=4, block_stride=2 * 2176, block_tokens=16, n_kv_heads=2, head_dim=128, bits=4)
    a.update(kw)
    return C.byref(N.QuantGeometry(*a.values()))


def lists(**kw):
    from ucmx import _native as N
    a = dict(offsets=FAKE, counts=0, block_ids=FAKE, positions=0, table=0, table_offsets=0, ctx_lens=0, n_req=1, total=3, table_size=0)
    a.update(kw)
    return C.byref(N.BlockLists(*a.values()))


def attend(**kw):
    from ucmx import _native as N
    a = dict(q=FAKE, q_stride=8 * 128, hq=8, q_offsets=0, n_tok=1, max_q=1, k=FAKE, kg=geom(), v=FAKE, vg=geom(), lists=lists(),
             scale=1.0, out=FAKE, lse=0, ws=FAKE, ws_bytes=1 << 40, stream=0)
    a.update(kw)
    return N.lib.ucmx_block_attention(*a.values())


@pytest.mark.parametrize("why", [
    dict(q=0), dict(out=0), dict(ws=0), dict(k=0), dict(v=0), dict(kg=None), dict(vg=None), dict(lists=None),
    dict(q=FAKE + 8), dict(out=FAKE + 2), dict(ws=FAKE + 4), dict(k=FAKE + 8), dict(q_stride=8 * 128 + 4), dict(q_stride=7 * 128),
    dict(hq=7), dict(hq=1), dict(hq=0), dict(max_q=0), dict(max_q=2), dict(max_q=2, q_offsets=FAKE), dict(n_tok=-1), dict(ws_bytes=64),
    "geom", "lists"])
def test_attention_refusals(why):
    from ucmx import _native as N
    if why == "geom":
        for kw in (dict(block_tokens=0), dict(n_kv_heads=0), dict(reserved=0), dict(token_stride=128), dict(token_stride=260),
                   dict(block_stride=4), dict(block_stride=-4096), dict(block_stride=0)):
            assert attend(kg=geom(**kw)) == N.EPARAM, kw
        assert attend(vg=geom(block_tokens=32)) == N.EPARAM
        for d in (32, 96, 120, 192, 512):
            x = dict(head_dim=d, token_stride=2 * d, block_stride=32 * d)
            assert attend(kg=geom(**x), vg=geom(**x), q_stride=8 * d) == N.EUNSUPPORTED
    elif why == "lists":
        for kw in (dict(offsets=0), dict(block_ids=0), dict(block_ids=0, positions=FAKE), dict(block_ids=0, positions=FAKE, table=FAKE),
                   dict(n_req=-1), dict(total=-1), dict(table_size=-1)):
            assert attend(lists=lists(**kw)) == N.EPARAM, kw
    else:
        assert attend(**why) == N.EPARAM
        assert N.last_error()


def test_nothing_to_do_is_fine():
    from ucmx import _native as N
    assert attend(lists=lists(n_req=0)) == N.OK
    assert attend(n_tok=0) == N.OK
    assert N.lib.ucmx_quant_write_tokens(None, None, 0, 0, 0, None, None, None, None) == N.OK
    assert N.lib.ucmx_quant_write_blocks(None, None, None, None, None, None, 0, None, None, None) == N.OK
    assert N.lib.ucmx_quant_read_blocks(None, None, None, None, 0, None, None, None, None, None) == N.OK


def test_quantised_cache_refusals():
    from ucmx import _native as N
    for kw in (dict(bits=2), dict(bits=16), dict(head_dim=96), dict(block_tokens=8), dict(block_tokens=24), dict(n_kv_heads=0)):
        assert N.lib.ucmx_quant_block_bytes(qgeom(**kw)) == 0, kw
        assert N.lib.ucmx_quant_write_tokens(FAKE, FAKE, 256, 256, 1, FAKE, FAKE, qgeom(**kw), None) == N.EUNSUPPORTED
    assert N.lib.ucmx_quant_block_bytes(qgeom()) == 2 * 2176
    assert N.lib.ucmx_quant_block_bytes(qgeom(bits=8, block_tokens=64)) == 2 * 4 * 4224
    w = lambda k=FAKE, v=FAKE, ks=256, vs=256, n=1, s=FAKE, c=FAKE, g=None: N.lib.ucmx_quant_write_tokens(  # noqa: E731
        k, v, ks, vs, n, s, c, g or qgeom(), None)
    for kw in (dict(k=0), dict(v=0), dict(s=0), dict(c=0), dict(k=FAKE + 2), dict(c=FAKE + 8), dict(ks=128), dict(vs=260), dict(n=-1),
               dict(g=qgeom(block_stride=2176)), dict(g=qgeom(block_stride=2 * 2176 + 8)), dict(g=qgeom(n_blocks=0))):
        assert w(**kw) == N.EPARAM, kw
    for kg in (geom(block_tokens=32), geom(n_kv_heads=1), geom(head_dim=64), geom(token_stride=260), geom(reserved=0), None):
        assert N.lib.ucmx_quant_write_blocks(FAKE, kg, FAKE, geom(), FAKE, None, 1, FAKE, qgeom(), None) == N.EPARAM
        assert N.lib.ucmx_quant_read_blocks(FAKE, qgeom(), FAKE, None, 1, FAKE, geom(), FAKE, kg, None) == N.EPARAM
    assert N.lib.ucmx_quant_write_blocks(FAKE, geom(), FAKE, geom(), None, None, 1, FAKE, qgeom(), None) == N.EPARAM
    assert N.lib.ucmx_quant_block_attention(FAKE, 1024, 8, None, 1, 1, None, qgeom(), lists(), 1.0, FAKE, None, FAKE, 1 << 40, None) == N.EPARAM
    assert N.lib.ucmx_quant_block_attention(FAKE, 1024, 8, None, 1, 1, FAKE, qgeom(bits=5), lists(), 1.0, FAKE, None, FAKE, 1 << 40,
                                            None) == N.EUNSUPPORTED
    assert N.lib.ucmx_attention_workspace_bytes(5, 8, 2, 128, 1) == 0
    assert N.lib.ucmx_attention_workspace_bytes(16, 8, 2, 96, 1) == 0
    assert N.lib.ucmx_attention_workspace_bytes(16, 8, 2, 128, 1) > 0


def test_python_front_refuses_what_it_can_see():
    from ucmx import ops
    with pytest.raises(ValueError):
        ops.QuantKvCache(torch.zeros((2, 2, 1, 2000), dtype=torch.uint8), head_dim=128, bits=4)
    with pytest.raises(ValueError):
        ops.QuantKvCache(torch.zeros((2, 2, 1, 2176), dtype=torch.int8), head_dim=128, bits=4)
    with pytest.raises(ValueError):
        ops.QuantKvCache.alloc(2, 24, 2, 128, 4, "cpu")
    c = ops.QuantKvCache.alloc(2, 32, 2, 128, 4, "cpu")
    assert c.block_bytes == 2 * 2 * 2176
    x = torch.zeros((1, 2, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.quant_write_tokens(c, x, x, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        ops.block_attention(x, x[None], x[None], torch.zeros(2, dtype=torch.int32), block_ids=torch.zeros(1, dtype=torch.int32))


def test_the_plain_form_packs_what_it_unpacks():
    for bits in (4, 8):
        for D in (64, 128, 256):
            g = torch.Generator().manual_seed(D + bits)
            k, v = (torch.randn((2, 32, 2, D), generator=g).to(torch.bfloat16) for _ in range(2))
            data = R.pack(k, v, bits)
            at = torch.cat([R.places(w, D, bits)[0].reshape(-1) for w in (0, 1)])
            assert sorted(set(at.tolist())) == list(range(32 * (D * bits // 8)))
            for (codes, scale, zero), x in zip(R.held(data, D, bits), (k, v)):
                c, s, z = R.to_codes(x, bits)
                assert torch.equal(codes, c) and torch.equal(scale, s) and torch.equal(zero, z)


def test_reading_back_into_blocks_that_lie_in_one_place():
    from ucmx import _native as N
    for kg, vg in ((geom(block_stride=0), geom()), (geom(), geom(block_stride=0))):
        assert N.lib.ucmx_quant_read_blocks(FAKE, qgeom(), FAKE, None, 1, FAKE, kg, FAKE, vg, None) == N.EPARAM


@pytest.mark.parametrize("quant", [False, True])
def test_numbers_beyond_32_bits_are_refused_by_the_python_front(quant):
    """Cut to 32 bits they would be other sizes: 2^32 + 1 query tokens per request one, 2^32 entries none."""
    from ucmx import ops
    from ucmx.retrieval import _fast
    cache = (FAKE, 4, 2 * 2176, 16, 2, 128, 4) if quant else (FAKE, 4096, 256, 16, 2, 128, 4) * 2
    call = _fast.quant_block_attention if quant else _fast.block_attention
    entry = ops._QUANT_BLOCK_ATTENTION if quant else ops._BLOCK_ATTENTION
    head = [FAKE, 1024, 8, 0, 1, 1]                                        # q, stride, heads, q_offsets, tokens, tokens per request
    lists = [FAKE, 0, FAKE, 0, 0, 0, 0, 1, 3, 0]
    tail = [1.0, FAKE, 0, FAKE, 64, 0]                                     # (a workspace of 64 bytes: never launched)
    assert call(entry, *head, *cache, *lists, *tail) < 0                   # EPARAM: the workspace is too small
    for which, at in ((head, 2), (head, 4), (head, 5), (lists, 7), (lists, 8), (lists, 9)):
        keep = which[at]
        which[at] = keep + 2 ** 32
        with pytest.raises(ValueError):
            call(entry, *head, *cache, *lists, *tail)
        which[at] = keep
    for at in range(3, 7):
        c = list(cache)
        c[at] += 2 ** 32
        with pytest.raises(ValueError):
            call(entry, *head, *c, *lists, *tail)
    with pytest.raises(ValueError):
        _fast.quant_write_tokens(ops._QUANT_WRITE_TOKENS, FAKE, FAKE, 256, 256, 0, FAKE, FAKE, 4, 4352, 16, 2 + 2 ** 32, 128, 4, 0)
